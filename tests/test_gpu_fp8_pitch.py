"""Answers of the 8-bit product whose rows lie on one, two and three elements (transmuter_amd/csrc/tmh_fp8.hip stores pairs of
columns where rows lie on pairs): odd widths in even pitches, and a first element off a pair. What lies between the
rows stays. Tolerances as in test_gpu_serving.py."""

import ctypes

import numpy as np
import pytest

import test_gpu_serving as base
from serving_plain import to_type, values
from transmuter_amd._lib import lib
from transmuter_amd.device import NX_TO_TMH
from transmuter_amd.serving import Fp8Weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("m,k,n", [(9, 400, 71), (100, 400, 71), (100, 272, 33), (300, 400, 301), (1024, 144, 1), (1030, 528, 2049)])
def test_rows_of_y(ctx, m, k, n, dtype):
    base.say("rows of y", m, k, n, dtype)
    rng = np.random.default_rng(m + k + n)
    a, sa = base.fp8_rows(rng, m, k)
    w, sw = base.fp8_weight(rng, n, k)
    at, st, weight = ctx.put(a, "f8_e4m3fn"), ctx.put(sa), Fp8Weight.prepare(ctx, w, sw)
    size = 4 if dtype == "f32" else 2
    for pitch in (n, n + 1, n + 3):
        for skip in (0, 1, 2):
            yt = ctx.put(to_type(np.full(m * pitch + skip, 7.0), dtype))
            ctx.check(lib().tmh_matmul_fp8(ctx.handle, weight.handle, at.ptr, m, k, st.ptr, None, 0,
                                           ctypes.c_void_p(yt.ptr.value + skip * size), NX_TO_TMH[dtype], pitch, None))
            y = yt.numpy()
            assert (values(y[:skip]) == 7).all()
            y = y[skip:].reshape(m, pitch)
            assert (values(y)[:, n:] == 7).all()
            base.check_product(y[:, :n], a, sa, w, sw, None, dtype)
