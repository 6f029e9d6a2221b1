"""Plain 64-bit implementations of the decoder-layer operators, and e4m3 in numpy."""

from __future__ import annotations

import numpy as np

from transmuter_amd.device import bf16_bits_to_f32, bf16_host, f32_to_bf16_bits

# Half a step of each type, relative to the value.
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f8": 2.0 ** -4}
# Half a step of each type's subnormal numbers, absolute.
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def _f8_table() -> np.ndarray:
    out = np.empty(256)
    for i in range(256):
        e, m = (i >> 3) & 15, i & 7
        v = np.nan if (e == 15 and m == 7) else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        out[i] = -v if i & 128 else v
    return out


F8 = _f8_table()


def f8_values(bits) -> np.ndarray:
    return F8[np.asarray(bits)]


def f8_bits(x) -> np.ndarray:
    """Values of magnitude up to 448 rounded to e4m3 (to nearest, ties to even)."""
    x = np.asarray(x, dtype=np.float64)
    mags = F8[:127]
    i = np.clip(np.searchsorted(mags, np.abs(x)), 1, 126)
    low = np.abs(x) - mags[i - 1]
    high = mags[i] - np.abs(x)
    i = np.where((low < high) | ((low == high) & ((i - 1) % 2 == 0)), i - 1, i)
    return (i | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def to_type(x, dtype):
    """f64 values as a host array of a float type."""
    x = np.asarray(x, dtype=np.float32)
    if dtype == "f32":
        return x
    return x.astype(np.float16) if dtype == "f16" else bf16_host(f32_to_bf16_bits(x))


def values(a) -> np.ndarray:
    """The f64 values of a float host array."""
    from transmuter_amd.device import BF16Host

    return (bf16_bits_to_f32(a) if isinstance(a, BF16Host) else np.asarray(a)).astype(np.float64)


def block_scales(y, floor=2.0 ** -126):
    """The scales [blocks, rows] of rows in 8 bits."""
    rows, cols = y.shape
    nb = -(-cols // 128)
    v = np.zeros((rows, nb * 128))
    v[:, :cols] = np.abs(y)
    top = v.reshape(rows, nb, 128).max(-1).T
    return np.where(top == 0, 1.0, np.maximum(top / 448, floor))


def expand(scales, cols):
    """[blocks, rows] scales for each of a row's columns, [rows, cols]."""
    return np.repeat(scales, 128, 0).T[:, :cols]


def rms_norm(x, gamma, residual=None, eps=1e-6):
    h = x if residual is None else x + residual
    return h, h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * gamma


def matmul(a, a_scales, w, w_scales, bias=None):
    """The products and the sums of their magnitudes."""
    n, k = w.shape
    x = a * expand(a_scales, k)
    v = w * np.repeat(np.repeat(w_scales, 128, 0), 128, 1)[:n, :k]
    y, mag = x @ v.T, np.abs(x) @ np.abs(v).T
    return (y, mag) if bias is None else (y + bias, mag + np.abs(bias))


def rotate(x, cos, sin, interleaved):
    """x [T, heads, dim]; cos, sin [T, rotary / 2]."""
    out, half = x.copy(), cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    first = (slice(0, 2 * half, 2) if interleaved else slice(0, half))
    second = (slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    out[..., first] = a * c - b * s
    out[..., second] = a * s + b * c
    return out


def attend(q, k_rows, v_rows, scale):
    """q [heads, dim] over k_rows, v_rows [tokens, kv_heads, dim]; also the sums of the weighted magnitudes."""
    heads, dim = q.shape
    tokens, kv_heads, _ = k_rows.shape
    if tokens == 0:
        return np.zeros_like(q), np.zeros_like(q)
    out, mag = np.empty_like(q), np.empty_like(q)
    for h in range(heads):
        g = h // (heads // kv_heads)
        s = scale * (k_rows[:, g] @ q[h])
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ v_rows[:, g]
        mag[h] = p @ np.abs(v_rows[:, g])
    return out, mag
