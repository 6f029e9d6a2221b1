"""Calls of more rows than one launch takes: the rows on both sides of the border are answered, and each once."""

import numpy as np
import pytest

from serving_plain import f8_values
from transmuter_amd import serving

pytestmark = pytest.mark.gpu


def test_norm_of_many_rows(ctx):
    """Rows of one column: y = x / sqrt(x^2 + eps), the sum into the residual's own memory (a row answered twice would be
    added to twice)."""
    t = 2 ** 26 + 77  # 2^24 workgroups and more
    print("norm of many rows", t, flush=True)
    x = np.resize(np.array([1.0, -2.0, 0.5, 4.0, -8.0], np.float16), (t, 1))
    xt, rt = ctx.put(x), ctx.put(np.resize(np.array([1.0, 2.0, -0.25], np.float16), (t, 1)))
    h = x.astype(np.float32) + np.resize(np.array([1.0, 2.0, -0.25], np.float32), (t, 1))
    y = ctx.empty((t, 1), "f16")
    out = serving.rms_norm(xt, ctx.put(np.ones(1, np.float16)), rt, eps=0.25, y=True, rows=False, out=serving.Norm(y, None, rt))
    assert np.array_equal(rt.numpy(), h.astype(np.float16))
    want = h / np.sqrt(h * h + np.float32(0.25))
    assert (np.abs(out.y.numpy() - want) <= 2.0 ** -10).all()
    for v in (xt, rt, y):
        v.free()


def test_quantize_many_rows(ctx):
    t = 2 ** 28 + 9  # blocks of 128, of which a workgroup takes 16
    print("quantize many rows", t, flush=True)
    x = np.resize(np.array([1.0, -2.0, 0.5, 448.0, -0.25, 0.0, 96.0], np.float16), (t, 1))
    xt = ctx.put(x)
    out = serving.quantize_rows(xt)
    xt.free()
    q, s = out.q.numpy(), out.scales.numpy()
    out.q.free(), out.scales.free()
    want = np.resize(np.array([448.0, -448.0, 448.0, 448.0, -448.0, 0.0, 448.0]), t)
    assert np.array_equal(f8_values(q[:, 0]), want)
    assert np.allclose(s[0], np.where(x[:, 0] == 0, 1, np.abs(x[:, 0].astype(np.float32)) / 448), rtol=2.0 ** -22, atol=0)
