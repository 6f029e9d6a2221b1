"""Rows in 8 bits of NaN and infinities, plain and behind a gate, and of gates of every size."""

import numpy as np
import pytest

import serving_plain as plain
from serving_plain import f8_values
from transmuter_amd import serving

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24


def test_nan_and_infinities(ctx):
    """A NaN makes its block's scale NaN, an infinity infinite; no other block has any of it."""
    print("quantize NaN and infinities", flush=True)
    x = np.full((5, 300), 2.0, np.float32)
    x[0, 3], x[1, 130], x[2, 299], x[3, 5], x[3, 6] = np.nan, np.inf, -np.inf, np.inf, np.nan
    out = serving.quantize_rows(ctx.put(x))
    q, s = f8_values(out.q.numpy()), out.scales.numpy()
    for row, block in ((0, 0), (3, 0)):
        assert np.isnan(s[block, row])
    assert s[1, 1] == np.inf and s[2, 2] == np.inf
    assert np.isnan(q[1, 130]) and (np.delete(q[1, 128:256], 2) == 0).all()
    assert np.isnan(q[2, 299]) and (q[2, 256:299] == 0).all()
    clean = np.ones((3, 5), bool)
    clean[0, 0] = clean[1, 1] = clean[2, 2] = clean[0, 3] = False
    assert (np.abs(s[clean] - 2 / 448) <= E32 * 2 / 448).all()
    assert (q[np.repeat(clean.T, 128, 1)[:, :300]] == 448).all()


@pytest.mark.parametrize("gate,up,scale,value", [
    (-np.inf, 1.0, np.nan, np.nan),   # -infinity * 0
    (np.inf, 1.0, np.inf, np.nan),    # an infinity, of an infinite scale
    (np.inf, 0.0, np.nan, np.nan),
    (np.nan, 1.0, np.nan, np.nan),
    (0.0, np.inf, np.nan, np.nan),    # 0 * an infinity
    (2.0, -np.inf, np.inf, np.nan),
    (-1e30, 1.0, None, 0.0),
    (-1e30, np.inf, np.nan, np.nan),  # 0 * an infinity
])
def test_gates(ctx, gate, up, scale, value):
    print("swiglu special", gate, up, flush=True)
    for n in (128, 100):  # rows on 16 bytes, and off them
        x = np.ones((2, 2 * n), np.float32)
        x[1, 7], x[1, n + 7] = gate, up
        out = serving.quantize_swiglu(ctx.put(x))
        q, s = f8_values(out.q.numpy()), out.scales.numpy()
        one = 1 / (1 + np.exp(-1.0))
        assert (np.abs(s[0, :1] - one / 448) <= 16 * E32 * one / 448).all()
        if scale is None:
            assert q[1, 7] == value and (np.abs(s[0, 1] - one / 448) <= 16 * E32 * one / 448)
        else:
            assert np.array_equal(s[0, 1], np.float32(scale), equal_nan=True)
            assert np.isnan(q[1, 7]) or np.isnan(scale)
            if scale == np.inf:
                assert (np.delete(q[1], 7) == 0).all()


def test_gates_of_every_size(ctx):
    """gate * sigmoid(gate), a block of 128 to each gate, from -88 (e^88 is within f32) to the largest numbers."""
    print("swiglu gates", flush=True)
    g = np.concatenate([np.linspace(-88, 20, 217), [1e3, 1e10, 1e37], -np.geomspace(1e-30, 1, 31), np.geomspace(1e-30, 1, 31)]).astype(np.float32)
    x = np.repeat(np.concatenate([g[:, None], np.ones((len(g), 1), np.float32)], 1), 128, 1)
    out = serving.quantize_swiglu(ctx.put(x))
    v = g.astype(np.float64)
    y = v / (1 + np.exp(-v))
    # The exponential's argument is rounded (128 log2 e at most, half a step of it: 2^-17 / 2, relatively as a factor), then
    # it, the sum, its reciprocal, the product with the gate and the scale by some steps more.
    tol = (2.0 ** -17 + 12 * E32) * np.abs(y)
    s = out.scales.numpy()[0].astype(np.float64)
    want = plain.block_scales(y[:, None])[0]
    assert (np.abs(s - want) <= tol / 448 + E32 * want).all()
    got = f8_values(out.q.numpy())[:, 5] * s
    fits = np.abs(y) >= 448 * 2.0 ** -126  # (below, the least scale's steps)
    assert (np.abs(got - y) <= tol * 2 + 4 * E32 * np.abs(y))[fits].all()
    assert (np.abs(got - y) <= 2.0 ** -4 * np.abs(y) + 2.0 ** -136).all()
