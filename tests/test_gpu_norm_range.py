"""The norm over the whole range of f32 and bf16: rows whose squares pass the largest number or fall below the smallest, with
an eps that counts, that does not, and none."""

import math

import numpy as np
import pytest

import serving_plain as plain
from serving_plain import HALF, TINY, to_type, values
from transmuter_amd import serving

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 64, 300, 2048, 12000, 40000])
@pytest.mark.parametrize("eps", [0.0, 1e-44, 1e-33, 1e-28, 1e-6, 1e30])
def test_rows_of_any_size(ctx, n, dtype, eps):
    print("norm range", n, dtype, eps, flush=True)
    rng = np.random.default_rng(n)
    exponents = [-147, -140, -126, -110, -100, -76, -64, -50, -40, -10, 0, 20, 50, 62, 65, 90, 110, 125]
    x = np.stack([(rng.random(n) + 0.5) * rng.choice([-1, 1], n) * 2.0 ** e for e in exponents])
    if n > 1:  # beside zeros, and beside far smaller ones
        x = np.concatenate([x, x * (rng.random(n) < 0.5), x * 2.0 ** rng.integers(-30, 1, n)])
        x[:, 0] = np.tile(2.0 ** np.array(exponents), 3)
    x = to_type(x, dtype)
    gamma = to_type(rng.random(n) + 0.5, dtype)
    eps = float(np.float32(eps))
    out = serving.rms_norm(ctx.put(x), ctx.put(gamma), eps=eps, y=True)
    with np.errstate(invalid="ignore"):
        _, y = plain.rms_norm(values(x), values(gamma), eps=eps)
    nothing = np.isnan(y).any(1)  # rows of zeros without eps (numbers that bf16 does not have): 0 / 0
    assert (nothing == (eps == 0) * ~values(x).any(1)).all()
    # The serial and tree sums, and a handful of single operations. Where y is subnormal, so is its product ahead of gamma
    # (up to 1.5), rounded to a step of f32's.
    extra = (8 * math.ceil(n / 2048) + 24) * E32
    got, s = values(out.y.numpy()), values(out.rows.scales.numpy())
    assert np.isnan(got[nothing]).all() and np.isnan(s[:, nothing]).all()
    got, y, s = got[~nothing], y[~nothing], s[:, ~nothing]
    assert (np.abs(got - y) <= (HALF[dtype] + extra) * np.abs(y) + TINY[dtype] + 1.5 * TINY["f32"]).all()
    want = plain.block_scales(y)
    # (A block whose values round to nothing in f32 may have the scale of zeros.)
    close = np.abs(s - want) <= (extra + 3 * E32) * want
    assert (close | ((s == 1) & (want <= 2.0 ** -126))).all()


@pytest.mark.parametrize("n", [300, 2048])
def test_zero_rows_without_eps(ctx, n):
    """0 / 0, as the formula has it; with an eps, however small, zeros."""
    print("norm of zeros", n, flush=True)
    x, gamma = ctx.put(np.zeros((2, n), np.float32)), ctx.put(np.ones(n, np.float32))
    assert np.isnan(serving.rms_norm(x, gamma, eps=0.0, y=True, rows=False).y.numpy()).all()
    for eps in (1e-44, 1e-30, 1e-6):
        assert (serving.rms_norm(x, gamma, eps=eps, y=True, rows=False).y.numpy() == 0).all()


def test_sum_of_rows_in_place(ctx):
    """The sum is h itself, whatever the squares were multiplied by."""
    print("norm range, sums", flush=True)
    rng = np.random.default_rng(3)
    for n in (100, 2048, 40000):
        x = ((rng.random((4, n)) + 0.5) * np.array([[2.0 ** -120], [2.0 ** -60], [1.0], [2.0 ** 120]])).astype(np.float32)
        r = (x * np.float32(0.25)).astype(np.float32)
        rt = ctx.put(r)
        out = serving.rms_norm(ctx.put(x), ctx.put(np.ones(n, np.float32)), rt, eps=0.0, out=serving.Norm(None, None, rt))
        assert np.array_equal(rt.numpy(), x + r) and out.sum is rt
