"""Attention of drafted steps at scores of any size, through each of its tiles and both ways in which parts of a sequence are joined, against 64
bits.

Tolerances: as test_gpu_drafts.check_draft has them, sums of half steps, but without what a score's own rounding may move (some 2^-22 of the
score), of which large scores leave nothing to be tested: here scores are equal bit for bit, or exact in f32."""

import math

import numpy as np
import pytest

import drafts_plain as drafts
import serving_plain as plain
from serving_plain import HALF, TINY, to_type, values
from test_gpu_drafts import E32, attend_tree, attend_tree_wide, draft_inputs, say

pytestmark = pytest.mark.gpu

SPLIT = {"f32": 0.0, "f16": 2.0 ** -20, "bf16": 2.0 ** -15}  # of a weight, what its two 16-bit parts leave out

# (length, nodes) of each sequence, heads, kv heads, dim, whether the table is wide; tiles of 16 columns, 64 and 128 (the rule is tree_form), of
# one worker's, of parts that meet in the kernel and of parts for the second one.
WAYS = {
    "16": ([(300, 9), (40, 5)], 4, 2, 128, False),
    "16 of many parts": ([(20000, 4)], 2, 1, 64, False),
    "16 whole": ([(30, 3)] * 700, 2, 1, 40, False),
    "64": ([(400, 16), (33, 9)], 4, 1, 128, True),
    "64 of many parts": ([(20000, 16)], 4, 1, 64, True),
    "64 whole": ([(50, 14)] * 600, 4, 1, 64, True),
    "128": ([(400, 40), (90, 7)], 4, 1, 128, True),
    "128 of many parts": ([(20000, 40)], 4, 1, 128, True),
    "128 whole": ([(50, 40)] * 300, 8, 2, 96, True),
    "64 of 256": ([(400, 16)], 4, 1, 256, True),
    "64 of 256 of many parts": ([(9000, 16)], 4, 1, 200, True),
}
TYPES = [("f16", w) for w in WAYS] + [("bf16", w) for w in WAYS] + [("f32", w) for w in WAYS if not WAYS[w][4]]


def sized(ctx, rng, way, dtype, kind):
    """The way's inputs, and a function that puts keys [pages, page, kv_heads, dim] in place and calls."""
    shapes, h, g, d, wide = WAYS[way]
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, 16, "token", dtype, kind)

    def call(q, keys, scale):
        bad = ~np.isfinite(k)  # (what lies past the sequences' ends stays)
        cache.k = ctx.put(to_type(np.where(bad, k, keys), dtype))
        cache.desc.k = cache.k.ptr
        return values((attend_tree_wide if wide else attend_tree)(ctx, cache, q, table, [n for n, _ in shapes], starts, mask, scale=scale).numpy())

    return shapes, h, g, d, k, v, table, starts, mask, call


def check(y, q, k, v, table, shapes, starts, mask, h, g, d, dtype, scale, delta):
    some = range(len(shapes)) if len(shapes) < 9 else (0, 1, len(shapes) // 2, len(shapes) - 1)
    for b in some:
        length, n = shapes[b]
        at = np.arange(length)
        for i in sorted({0, 1, n // 2, n - 1}):
            r = starts[b] + i
            seen = drafts.sees(None if mask is None else mask[r], i, n, length, 0)
            where = (table[b, at[seen] // 16], at[seen] % 16)
            want, mag = plain.attend(q[r].reshape(h, d), k[where], v[where], scale)
            tol = mag * (4 * delta + SPLIT[dtype] + (seen.sum() / 64 + 200) * E32) + HALF[dtype] * np.abs(want) + 4 * TINY[dtype]
            got = y[r].reshape(h, d)
            bad = ~(np.abs(got - want) <= tol)
            assert not bad.any(), (b, i, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


@pytest.mark.parametrize("dtype,way", TYPES)
def test_scores_of_any_size(ctx, dtype, way):
    """Some tokens' keys alike and far ahead of all others' (or, of queries of the other sign, behind them, the others alike): the leaders weigh the
    same, the rest nothing (scores are 10000 and more apart)."""
    say("scores of any size", dtype, way)
    rng = np.random.default_rng(len(way))
    kind = "chain" if "whole" in way else "tree"
    shapes, h, g, d, k, v, table, starts, mask, call = sized(ctx, rng, way, dtype, kind)
    sizes = [50, 300, 2000, 3000, 8000, 20000, 60000] if dtype == "f16" else [50, 3000, 1e4, 3e4, 1e5, 1e8, 1e12, 1e17]
    sign = rng.choice([-1.0, 1.0], d)
    ahead = np.where(rng.random(k.shape[:2]) < 0.1, 1.0, 0.5)[:, :, None, None] * np.ones((1, 1, g, 1))
    t, scale = int(starts[-1]), 1 / math.sqrt(d)
    of_head = rng.choice([1.0, 0.5, 1.0, -1.0], (t, h, 1))
    for size in sizes:
        c = values(to_type(np.array([size]), "bf16" if dtype == "f32" else dtype))[0]  # (few bits: products are exact in 64)
        keys = c * ahead * sign
        q = to_type((c * of_head * sign).reshape(t, h * d), dtype)
        for s in (scale, -scale):
            say("size", size, s)
            check(call(q, keys, s), values(q), keys, v, table, shapes, starts, mask, h, g, d, dtype, s, 0.0)


@pytest.mark.parametrize("base", [2.0 ** 10, 2.0 ** 22, -2.0 ** 22])
@pytest.mark.parametrize("dtype,way", [(t, w) for t, w in TYPES if WAYS[w][4]])
def test_large_scores_near_each_other(ctx, dtype, way, base):
    """Scores of about `base` that differ by whole numbers up to 16, exact in f32: their differences are, and make the weights. (Tiles of 16 round
    a score times its scale first, to f32, as attention of one token does.)"""
    say("scores near each other", dtype, way, base)
    rng = np.random.default_rng(len(way) + 7)
    shapes, h, g, d, k, v, table, starts, mask, call = sized(ctx, rng, way, dtype, "tree")
    keys = np.zeros(k.shape)
    keys[..., 0] = math.copysign(math.sqrt(abs(base)), base)
    keys[..., 1] = rng.integers(0, 9, k.shape[:3])
    t = int(starts[-1])
    q = np.zeros((t, h, d))
    q[..., 0], q[..., 1] = math.sqrt(abs(base)), rng.choice([1, 2, -1], (t, h))
    q = to_type(q.reshape(t, h * d), dtype)
    # A difference, up to 24 in base-2 logarithms, by the scale, itself rounded twice (half a step each), the sum with the factor's exponent (up to
    # 64), the exponential's two half steps.
    delta = 24 * 3 * E32 + 64 * E32 + 4 * E32
    check(call(q, keys, 1.0), values(q), keys, v, table, shapes, starts, mask, h, g, d, dtype, 1.0, delta)
