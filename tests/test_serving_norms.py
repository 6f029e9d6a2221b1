"""The 2-norm bounds of serving_norms.py on the host: models of right arithmetic are within them, and models that lose what the
kernels keep (the 8-bit unit's cuts in an f32 product, one 16-bit part of a weight instead of two) are not."""

import numpy as np
import pytest

import serving_norms as norms
from serving_plain import expand, f8_bits, f8_values, to_type, values

PRODUCTS = [(40, 384, 50), (40, 512, 70), (33, 1040, 64), (64, 2048, 96), (16, 4096, 130), (17, 11008, 40)]


def inputs(m, k, n):
    rng = np.random.default_rng(m + k + n)
    a = f8_values(f8_bits(np.clip(rng.standard_normal((m, k)) * 100, -448, 448)))
    w = f8_values(f8_bits(np.clip(rng.standard_normal((n, k)) * 100, -448, 448)))
    return a, (rng.random((-(-k // 128), m)) + 0.2).astype(np.float32) * 0.01, w, (rng.random((-(-n // 128), -(-k // 128))) + 0.2).astype(np.float32) * 1e-3


def blocks_of(a, sa, w, sw, eight):
    """The product in f32, block by block of 128, each of sums `eight` of eight products."""
    m, k = a.shape
    n = len(w)
    y = np.zeros((m, n), np.float32)
    for b in range(-(-k // 128)):
        x, v = a[:, 128 * b:128 * b + 128], w[:, 128 * b:128 * b + 128]
        c = np.zeros((m, n), np.float32)
        for i in range(0, x.shape[1], 8):
            c = (c + eight(x[:, None, i:i + 8] * v[None, :, i:i + 8])).astype(np.float32)
        s = (sa[b][:, None].astype(np.float32) * np.repeat(sw[:, b], 128)[:n].astype(np.float32)).astype(np.float32)
        y = (y + c * s).astype(np.float32)
    return y.astype(np.float64)


@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_product(m, k, n):
    a, sa, w, sw = inputs(m, k, n)
    want, spread = norms.product(a, sa.astype(np.float64), w, sw.astype(np.float64))
    bound = norms.product_bound(want, spread, k, "f32")
    assert bound < 5e-6 * norms.norm(want)
    assert norms.norm(blocks_of(a, sa, w, sw, lambda p: p.sum(-1)) - want) <= bound

    def cut(p):
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(p).max(-1, keepdims=True), 1e-30))) - 13)
        return (np.trunc(p / step) * step).sum(-1)

    assert norms.norm(blocks_of(a, sa, w, sw, cut) - want) > 2 * bound


def split(p, dtype, both):
    """Weights (at most 1) as a kernel's 16-bit parts hold them."""
    x = np.asarray(p, np.float32) * np.float32(2.0 ** 15 if dtype == "f16" else 1)
    if dtype == "f16":
        hi = x.astype(np.float16).astype(np.float32)
        lo = (x - hi).astype(np.float16).astype(np.float32)
    else:
        hi = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        lo = values(to_type(x - hi, "bf16"))
    return (hi.astype(np.float64) + (lo if both else 0)) / (2.0 ** 15 if dtype == "f16" else 1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,dim", [(40, 4, 64), (100, 8, 128), (300, 16, 128), (700, 16, 64), (1000, 8, 96), (2000, 4, 128),
                                              (5000, 4, 256), (9000, 2, 128)])
def test_attention(tokens, heads, dim, dtype):
    rng = np.random.default_rng(tokens + dim)
    q, k, v = (values(to_type(rng.standard_normal(s), dtype)) for s in ((heads, dim), (tokens, 1, dim), (tokens, 1, dim)))
    scale = dim ** -0.5
    want, spread, rms, largest = norms.attention(q, k, v, scale)
    bound = norms.attention_bound(want, spread, rms, largest, tokens, dtype)
    parts = "f16" if dtype == "f32" else dtype

    def model(both):
        s = (k[:, 0].astype(np.float32) @ q.T.astype(np.float32)) * np.float32(scale)
        p = np.exp(s - s.max(0)).astype(np.float32)
        kept = p.astype(np.float64) if dtype == "f32" and both else split(p, parts, both)
        y = (kept.T @ v[:, 0]) / p.sum(0, dtype=np.float64)[:, None]
        return values(to_type(y, dtype))

    assert norms.norm(model(True) - want) <= bound
    assert norms.norm(model(False) - want) > bound
