"""The 8-bit product at sizes that reach each of its kernels and launch shapes (transmuter_amd/csrc/tmh_fp8.hip,
plan_of), ragged in every direction, against the plain 64-bit product. Tolerances as in test_gpu_serving.py."""

import ctypes

import numpy as np
import pytest

import test_gpu_serving as base
from serving_plain import to_type, values
from transmuter_amd import _lib, serving
from transmuter_amd._lib import lib
from transmuter_amd.device import NX_TO_TMH
from transmuter_amd.serving import Fp8Weight, Rows8

pytestmark = pytest.mark.gpu

# Rows by 16 and 32 (one and two column tiles), by 64 in one group and in several, and each shape of tile, whole and in
# parts of K; K of one block, of an odd and an even number of them, ending inside one.
SHAPES = [(16, 272, 530), (20, 400, 16401), (32, 2064, 16500), (33, 4112, 100), (64, 1936, 31), (65, 272, 40),
          (100, 400, 333), (190, 528, 70), (130, 128, 1100), (66, 3984, 4000), (300, 5008, 130), (1024, 144, 2048),
          (1000, 400, 2001), (1000, 8208, 301), (515, 144, 22001), (2050, 144, 12301), (1300, 656, 5003), (2100, 272, 21001)]


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_launch_shapes(ctx, m, k, n, dtype):
    base.say("launch shape", m, k, n, dtype)
    rng = np.random.default_rng(m + 5 * k + n)
    a, sa = base.fp8_rows(rng, m, k)
    w, sw = base.fp8_weight(rng, n, k)
    bias = to_type(rng.standard_normal(n), dtype) if (m + n) % 2 else None
    y = serving.matmul_fp8(Rows8(ctx.put(a, "f8_e4m3fn"), ctx.put(sa)), Fp8Weight.prepare(ctx, w, sw),
                           ctx.put(bias) if bias is not None else None, y_type=dtype)
    base.check_product(y.numpy(), a, sa, w, sw, values(bias) if bias is not None else None, dtype)


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("m,k,n", [(9, 400, 70), (30, 400, 70), (60, 1040, 70), (100, 400, 70), (100, 5008, 70), (1024, 144, 300)])
def test_pitches(ctx, m, k, n, dtype):
    """Rows of A with NaN bytes between them (in reach of a load of whole blocks), a pitch of Y that is no multiple of a
    store: neither shows."""
    base.say("pitches", m, k, n, dtype)
    rng = np.random.default_rng(m + k)
    a, sa = base.fp8_rows(rng, m, k)
    wide = np.full((m, k + 112), 0x7F, np.uint8)
    wide[:, :k] = a
    w, sw = base.fp8_weight(rng, n, k)
    at, st, weight = ctx.put(wide, "f8_e4m3fn"), ctx.put(sa), Fp8Weight.prepare(ctx, w, sw)
    for pitch in (n, n + 2, n + 5):
        yt = ctx.put(to_type(np.full((m, pitch), 7.0), dtype))
        ctx.check(lib().tmh_matmul_fp8(ctx.handle, weight.handle, at.ptr, m, k + 112, st.ptr, None, 0, yt.ptr, NX_TO_TMH[dtype], pitch, None))
        y = yt.numpy()
        assert (values(y)[:, n:] == 7).all()
        base.check_product(y[:, :n], a, sa, w, sw, None, dtype)


@pytest.mark.parametrize("m", [16, 32, 64, 200])
def test_rows_of_nan_stay_their_own(ctx, m):
    """Every other row of A is NaN bytes: the rows between them, and rows past the last, have none of it."""
    base.say("rows of nan", m)
    rng = np.random.default_rng(m)
    k, n = 272, 140
    a, sa = base.fp8_rows(rng, m - 1, k)
    a[1::2] = 0x7F
    flat = np.concatenate([a, np.full((1, k), 0x7F, np.uint8)])  # a row behind the last that the call does not name
    w, sw = base.fp8_weight(rng, n, k)
    at, st, weight = ctx.put(flat, "f8_e4m3fn"), ctx.put(sa), Fp8Weight.prepare(ctx, w, sw)
    for dtype in ("f16", "f32"):
        yt = ctx.empty((m - 1, n), dtype)
        ctx.check(lib().tmh_matmul_fp8(ctx.handle, weight.handle, at.ptr, m - 1, k, st.ptr, None, 0, yt.ptr, NX_TO_TMH[dtype], n, None))
        y = yt.numpy()
        assert np.isnan(y[1::2]).all()
        base.check_product(y[0::2], a[0::2], sa[:, 0::2], w, sw, None, dtype)


def test_parts_need_the_workspace_before_a_capture():
    """A product in parts of K on a fresh context inside a capture is refused, and runs once it ran outside."""
    from transmuter_amd import Context

    base.say("parts in a capture")
    c = Context(0)
    try:
        rng = np.random.default_rng(1)
        m, k, n = 1000, 8192, 300
        a, sa = base.fp8_rows(rng, m, k)
        w, sw = base.fp8_weight(rng, n, k)
        weight, at, st, y = Fp8Weight.prepare(c, w, sw), c.put(a, "f8_e4m3fn"), c.put(sa), c.empty((m, n), "f16")

        def call():
            return lib().tmh_matmul_fp8(c.handle, weight.handle, at.ptr, m, k, st.ptr, None, 0, y.ptr, _lib.F16, n, None)

        def capture():
            c.check(lib().tmh_graph_begin(c.handle, None))
            status = call()
            graph = ctypes.c_void_p()
            c.check(lib().tmh_graph_end(c.handle, None, ctypes.byref(graph)))
            return status, graph

        status, graph = capture()
        c.check(lib().tmh_graph_destroy(c.handle, graph))
        assert status == _lib.ERR_UNSUPPORTED and b"before the capture" in lib().tmh_last_error(c.handle)
        c.check(call())
        want = y.numpy().copy()
        base.check_product(want, a, sa, w, sw, None, "f16")
        status, graph = capture()
        assert status == _lib.OK
        for _ in range(3):
            c.check(lib().tmh_upload(c.handle, y.ptr, np.zeros((m, n), np.float16).ctypes.data_as(ctypes.c_void_p), 2 * m * n))
            c.check(lib().tmh_graph_launch(c.handle, graph, None))
            assert np.array_equal(y.numpy(), want)
            c.check(call())
        c.synchronize()
        c.check(lib().tmh_graph_destroy(c.handle, graph))
    finally:
        c.close()
