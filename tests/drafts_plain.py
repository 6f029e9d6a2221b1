"""Plain 64-bit implementations of the operators of a drafted step: what a row of a tree sees, attention over it, and tokens
drawn from logits."""

from __future__ import annotations

import numpy as np

import serving_plain as plain

LEAST = 2.0 ** -44


def head_norm(x, gamma, eps):
    """x [T, heads, dim] normed over each head."""
    with np.errstate(invalid="ignore"):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma


def random_tree(rng, n, words, reach=8, whole=True):
    """The masks [n, words] of a tree of n nodes, each the child of one of the `reach` before it; with whole false bits are
    taken out at random, rows without any among them."""
    seen = np.zeros((n, 64 * words), bool)
    for i in range(n):
        if i:
            seen[i] = seen[rng.integers(max(0, i - reach), i)]
        if i < 64 * words:
            seen[i, i] = True
    if not whole:
        seen &= rng.random(seen.shape) < 0.6
        seen[rng.random(n) < 0.3] = False
    return pack(seen)


def pack(seen):
    """Bits [rows, 64 * words] as s64 words."""
    return np.packbits(seen, axis=-1, bitorder="little").view("<i8").reshape(len(seen), seen.shape[1] // 64)


def sees(mask, i, n, length, window):
    """The tokens [length] that node i of n sees: `mask` its row's words, or None (a chain)."""
    first = length - n
    out = np.zeros(length, bool)
    out[:max(first, 0)] = True
    bits = np.arange(n) <= i if mask is None else np.unpackbits(np.asarray(mask).astype("<i8").view(np.uint8), bitorder="little")
    for j in range(n):
        if first + j >= 0:
            out[first + j] = j < len(bits) and bits[j]
    if window:
        out[np.flatnonzero(out)[:-window]] = False
    return out


def sample(row, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """The token drawn from one row of logits (f64)."""
    row = np.where(np.isnan(row), -np.inf, row)
    top = row.max()
    if top == -np.inf:
        return -1
    if not temperature > 0:
        return int(np.flatnonzero(row == top)[0])
    if top == np.inf:
        w = (row == np.inf).astype(np.float64)
    else:
        with np.errstate(invalid="ignore", under="ignore"):
            w = np.exp((row - top) / temperature)
        w[row == -np.inf] = 0
    w[w < LEAST] = 0
    order = np.argsort(-row, kind="stable")
    if 0 < top_k < len(row):
        order = order[:top_k]
    if top_p < 1:
        sums = np.cumsum(w[order])
        order = order[:1 + np.searchsorted(sums, top_p * sums[-1])]
    if min_p > 0:
        order = order[w[order] >= min(min_p, 1.0)]
    order = np.sort(order[w[order] > 0])
    sums = np.cumsum(w[order])
    at = np.searchsorted(sums, u * sums[-1], side="right")
    return int(order[min(at, len(order) - 1)])


def attend(q, k, v, seen, scale):
    """q [heads, dim] over those of k, v [tokens, kv_heads, dim] that are seen; also the weighted magnitudes."""
    return plain.attend(q, k[seen], v[seen], scale)
