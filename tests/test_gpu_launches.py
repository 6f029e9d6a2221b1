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


def test_product_of_many_unaligned_rows():
    """More 16-byte pieces of rows off 16 bytes than one launch copies: 2^22 rows of 16385 bytes (64 times the same 2^16)."""
    import ctypes

    from serving_plain import expand, f8_bits
    from transmuter_amd import Context, _lib
    from transmuter_amd._lib import lib

    k, n, rows, times = 16385, 16, 2 ** 16, 64
    print("product of many rows", rows * times, k, n, flush=True)
    c = Context(0)
    try:
        rng = np.random.default_rng(0)
        a = rng.integers(0, 0x70, (rows, k), np.uint8)
        w = f8_bits(np.clip(rng.standard_normal((n, k)) * 100, -448, 448))
        sw = np.full((1, -(-k // 128)), 2.0 ** -10, np.float32)
        weight = serving.Fp8Weight.prepare(c, w, sw)
        sa = c.put(np.ones((-(-k // 128), rows * times), np.float32))
        at, y = c.empty((rows * times, k), "f8_e4m3fn"), c.empty((rows * times, n), "f32")
        for i in range(times):
            c.check(lib().tmh_upload(c.handle, ctypes.c_void_p(at.ptr.value + i * a.nbytes), a.ctypes.data_as(ctypes.c_void_p), a.nbytes))
        c.check(lib().tmh_matmul_fp8(c.handle, weight.handle, at.ptr, rows * times, k, sa.ptr, None, 0, y.ptr, _lib.F32, n, None))
        got = y.numpy().reshape(times, rows, n)
        assert (got == got[:1]).all()
        some = [0, 1, 2, 77, rows - 1]
        x, v = f8_values(a[some]), f8_values(w) * expand(np.repeat(sw.astype(np.float64), n, 0).T, k)
        want, mag = x @ v.T, np.abs(x) @ np.abs(v).T
        assert (np.abs(got[0][some] - want) <= (128 + 129 + 24) * 2.0 ** -23 * mag).all()
        for t in (at, y, sa):
            t.free()
        weight.free()
    finally:
        c.close()
