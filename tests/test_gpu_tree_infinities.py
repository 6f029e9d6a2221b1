"""Infinities and NaN in attention of drafted steps, through each of its tiles and both ways in which parts of a sequence are joined."""

import math

import numpy as np
import pytest

from serving_plain import HALF, TINY, to_type, values
from test_gpu_drafts import E32, attend_tree, attend_tree_wide, draft_inputs, say
from test_gpu_tree_scores import SPLIT, TYPES, WAYS

pytestmark = pytest.mark.gpu


def put(ctx, cache, keys, vals, dtype):
    cache.k, cache.v = ctx.put(to_type(keys, dtype)), ctx.put(to_type(vals, dtype))
    cache.desc.k, cache.desc.v = cache.k.ptr, cache.v.ptr


@pytest.mark.parametrize("dtype,way", TYPES)
def test_infinity_of_any_weight(ctx, dtype, way):
    """An infinity that all rows see, at a weight of 2^-w of the largest, w up to 90, is one of its sign in their answers; the other
    dimensions answer as without."""
    say("infinity of any weight", dtype, way)
    rng = np.random.default_rng(len(way))
    shapes, h, g, d, wide = WAYS[way]
    shapes = [(n, m) for n, m in shapes if n > m]
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, 16, "token", dtype, "chain")
    run, t = attend_tree_wide if wide else attend_tree, int(starts[-1])
    lengths = [n for n, _ in shapes]
    # Of each sequence a token ahead of the step's own; every other one of the rest is of the largest weight.
    at = np.array([rng.integers(0, n - m) for n, m in shapes])
    place = np.array([table[b, i // 16] for b, i in enumerate(at)]), at % 16
    score = np.where(rng.permutation(16) % 2, 0.0, -250.0)[None, :, None] * np.ones(k.shape[:3])
    q = np.zeros((t, h, d))
    q[..., 0] = 1
    q = to_type(q.reshape(t, h * d), dtype)
    for w in (1, 20, 37, 38, 39, 45, 63, 80, 89):
        say("weight", w)
        score[place] = -w
        keys, vals = np.where(np.isfinite(k), 0.0, k), v.copy()
        keys[..., 0] = np.where(np.isfinite(k[..., 0]), score, k[..., 0])
        vals[place[0], place[1], :, 1::3] = np.inf
        vals[place[0], place[1], :, 2::3] = -np.inf
        put(ctx, cache, keys, vals, dtype)
        got = values(run(ctx, cache, q, table, lengths, starts, None, scale=math.log(2)).numpy()).reshape(t, h, d)
        assert (got[..., 1::3] == np.inf).all() and (got[..., 2::3] == -np.inf).all(), w
        for b in range(len(shapes)) if len(shapes) < 9 else (0, 1, len(shapes) - 1):
            for i in (0, shapes[b][1] - 1):
                tokens = np.arange(lengths[b] - shapes[b][1] + i + 1)
                where = table[b, tokens // 16], tokens % 16
                weights = 2.0 ** score[where][:, 0]
                weights /= weights.sum()
                of_v = vals[where][..., ::3]
                want = np.repeat(np.einsum("t,tgd->gd", weights, of_v), h // g, axis=0)
                mag = np.repeat(np.einsum("t,tgd->gd", weights, np.abs(of_v)), h // g, axis=0)
                # (A score's roundings, of the scale's two by up to 90 and its own, move a weight by 90 * 3 half steps at most.)
                tol = HALF[dtype] * np.abs(want) + mag * (SPLIT[dtype] + 2 * 270 * E32 + (len(tokens) / 64 + 200) * E32) + 4 * TINY[dtype]
                assert (np.abs(got[starts[b] + i][:, ::3] - want) <= tol).all(), (w, b, i)
