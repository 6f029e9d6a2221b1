"""Bounds in the 2-norm for the decoder-layer operators that multiply: what the roundings of a right answer come to together,
where a bound on each element has to allow for all of them meeting in one.

A sum of n terms in f32 is off by a random walk of n roundings: sqrt(n) steps of the partial sums, whose size is that of the
root of the terms' squares' sum (`spread` below) for terms of either sign. Rounding the answer to its own type is known
(the distance of the exact answer to its rounding); beside it an error e ahead of it moves the answer by 2 e at most."""

import numpy as np

from serving_plain import expand, to_type, values

STEP = 2.0 ** -23  # of f32 (a cut; half of it a rounding)


def norm(x) -> float:
    return float(np.linalg.norm(np.asarray(x, np.float64)))


def rounded(want, dtype):
    """What rounding the exact answer to its type leaves."""
    return 0.0 if dtype == "f32" else norm(values(to_type(want, dtype)) - want)


def product(a, a_scales, w, w_scales):
    """The 64-bit product of values and scales, and the spread of its terms."""
    k, n = a.shape[1], w.shape[0]
    x = a * expand(a_scales, k)
    v = w * np.repeat(np.repeat(w_scales, 128, 0), 128, 1)[:n, :k]
    return x @ v.T, np.sqrt((x * x) @ (v * v).T)


def product_bound(want, spread, k, dtype):
    """An f32 answer: products are exact; a block of 128 is sixteen sums of eight of them, cut, and the blocks' sums are added
    with two products of scales. The 8-bit unit's cuts, behind a 16-bit answer, are up to 5e-5 of the answer by
    what the header states."""
    blocks = -(-k // 128)
    e = (16 * STEP + np.sqrt(blocks) * STEP / 2 + 4 * STEP / 2) * norm(spread)
    if dtype == "f32":
        return e
    return rounded(want, dtype) + 2 * (e + 5e-5 * norm(spread))


def attention(q, k, v, scale):
    """The 64-bit answer of q [heads, dim] over k, v [tokens, kv_heads, dim], the spread of its terms, and the scores'
    root mean square and largest magnitude."""
    heads = len(q)
    group = heads // k.shape[1]
    want, spread, scores = np.empty_like(q), np.empty_like(q), []
    for h in range(heads):
        s = scale * (k[:, h // group] @ q[h])
        p = np.exp(s - s.max())
        p /= p.sum()
        want[h], spread[h] = p @ v[:, h // group], np.sqrt((p * p) @ (v[:, h // group] ** 2))
        scores.append(s)
    scores = np.array(scores)
    return want, spread, float(np.sqrt((scores ** 2).mean())), float(np.abs(scores).max())


# What the two 16-bit parts of a weight leave of it, relatively.
PARTS = {"f32": 0.0, "f16": 2.0 ** -21, "bf16": 2.0 ** -16}


def attention_bound(want, spread, rms, largest, tokens, dtype):
    """A score is a sum of dim products (partial sums of the scores' size) and two products more, a weight its exponential
    (two steps); then the weights' and the values' sums over the tokens."""
    dim = want.shape[1]
    e = (np.sqrt(dim) * 2 * STEP * rms + 2 * STEP * largest + 4 * STEP + np.sqrt(tokens) * STEP + PARTS[dtype]) * norm(spread)
    return rounded(want, dtype) + (e if dtype == "f32" else 2 * e)
