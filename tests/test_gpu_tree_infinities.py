"""Infinities and NaN in attention of drafted steps, through each of its tiles and both ways in which parts of a sequence are joined."""

import math
import time

import numpy as np
import pytest

import drafts_plain as drafts
import serving_plain as plain
from serving_plain import HALF, TINY, to_type, values
from test_gpu_drafts import E32, attend_tree, attend_tree_wide, draft_inputs, say
from test_gpu_drafts import check_draft
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


def some_rows(shapes, without=()):
    """Pairs of sequence and node."""
    b = range(len(shapes)) if len(shapes) < 9 else (0, 1, len(shapes) - 1)
    return {(i, j) for i in b for j in (0, 1, shapes[i][1] // 2, shapes[i][1] - 1)} - set(without)


@pytest.mark.parametrize("dtype,way", TYPES)
def test_a_query_of_nan_costs_its_row(ctx, dtype, way):
    """Some rows' queries with a NaN: their heads answer NaN, all others as ever, and the call takes no longer (done again, the columns of
    their tiles take a hundred times as long and more)."""
    say("query of NaN", dtype, way)
    rng = np.random.default_rng(len(way) + 1)
    shapes, h, g, d, wide = WAYS[way]
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, 16, "token", dtype, "tree")
    run = attend_tree_wide if wide else attend_tree
    lengths, scale = [n for n, _ in shapes], 1 / math.sqrt(d)
    bad = values(q)
    nan = [(b, m - 1) for b, (_, m) in enumerate(shapes)]
    for b, i in nan:
        bad[starts[b] + i, 3] = np.nan  # of the first head
    bad = to_type(bad, dtype)
    got = run(ctx, cache, bad, table, lengths, starts, mask).numpy()
    check_draft(got, q, k, v, table, shapes, starts, mask, 16, h, g, d, dtype, scale, rows=some_rows(shapes, nan))
    rows = np.array([starts[b] + i for b, i in nan])
    assert np.isnan(values(got)[rows, :d]).all() and (h == 1 or np.isfinite(values(got)[rows, d:]).all())
    width = 10 ** 6 // 16 if wide else table.shape[1]
    dev = ctx.put(np.pad(table, ((0, 0), (0, width - table.shape[1])), constant_values=-1)), ctx.put(np.asarray(lengths, np.int32)), ctx.put(starts), ctx.put(mask)
    took = []
    for x in (ctx.put(q), ctx.put(bad)):
        out = ctx.empty(q.shape, dtype)
        each = []
        for _ in range(6):
            ctx.synchronize()
            begin = time.perf_counter()
            for _ in range(10):
                cache.attend_tree(x, *dev, out=out)
            ctx.synchronize()
            each.append(time.perf_counter() - begin)
        took.append(min(each))
    say("us", [t * 1e5 for t in took])
    assert took[1] < 5 * took[0]


@pytest.mark.parametrize("dtype,way", TYPES)
def test_values_that_some_rows_see(ctx, dtype, way):
    """NaN and infinities in a few dimensions of two tokens, one that all rows see and a node of the step's own: in those dimensions the rows that see them
    answer with them, and in the others, as rows that do not see them in all, as without."""
    say("values that some rows see", dtype, way)
    rng = np.random.default_rng(len(way) + 2)
    shapes, h, g, d, wide = WAYS[way]
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, 16, "token", dtype, "tree")
    run = attend_tree_wide if wide else attend_tree
    lengths = [n for n, _ in shapes]
    vals, clean = v.copy(), v.copy()
    for b, (n, m) in enumerate(shapes):
        for at, dims in ((int(rng.integers(0, n - m)), (2, 9)), (n - m + 1, (5, 11))):
            where = table[b, at // 16], at % 16
            vals[where][:, dims[0]], vals[where][:, dims[1]] = np.nan, np.inf
            clean[where][:, dims] = 0
    put(ctx, cache, k, vals, dtype)
    got = values(run(ctx, cache, q, table, lengths, starts, mask).numpy()).reshape(-1, h, d).copy()
    node_seen = np.unpackbits(mask.astype("<i8").view(np.uint8), axis=-1, bitorder="little")[:, 1].astype(bool)
    assert np.isnan(got[..., 2]).all() and (got[..., 9] == np.inf).all()
    assert np.isnan(got[node_seen][..., 5]).all() and (got[node_seen][..., 11] == np.inf).all()
    assert np.isfinite(got[~node_seen][..., [5, 11]]).all()
    # The rest against the 64-bit form, in whose place of those dimensions are zeros.
    rows = some_rows(shapes)
    for b, i in rows:
        r, (n, m) = starts[b] + i, shapes[b]
        tokens = np.flatnonzero(drafts.sees(mask[r], i, m, n, 0))
        where = table[b, tokens // 16], tokens % 16
        want, _ = plain.attend(values(q)[r].reshape(h, d), k[where], clean[where], 1 / math.sqrt(d))
        special = [2, 9] + [5, 11] * bool(node_seen[r])
        got[r][:, special] = want[:, special]
    check_draft(got.reshape(len(q), -1), q, k, clean, table, shapes, starts, mask, 16, h, g, d, dtype, 1 / math.sqrt(d), rows=rows)


@pytest.mark.parametrize("dtype,way", TYPES)
def test_values_that_some_windows_leave(ctx, dtype, way):
    """A NaN in a value of a token that is in some rows' windows and before others', which answer as without it."""
    say("values that some windows leave", dtype, way)
    rng = np.random.default_rng(len(way) + 3)
    shapes, h, g, d, wide = WAYS[way]
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, 16, "token", dtype, "tree")
    run = attend_tree_wide if wide else attend_tree
    lengths, window, left = [n for n, _ in shapes], 12, {}
    vals = v.copy()
    for b, (n, m) in enumerate(shapes):
        at = n - m - min(9, n - m)
        vals[table[b, at // 16], at % 16, :, 3] = np.nan
        left[b] = at
    put(ctx, cache, k, vals, dtype)
    y = run(ctx, cache, q, table, lengths, starts, mask, window=window).numpy()
    got, clean = values(y).reshape(-1, h, d), []
    for b, (n, m) in enumerate(shapes):
        for i in range(m):
            if drafts.sees(mask[starts[b] + i], i, m, n, window)[left[b]]:
                assert np.isnan(got[starts[b] + i, :, 3]).all() and np.isfinite(got[starts[b] + i, :, 4:]).all()
            else:
                clean.append((b, i))
                assert np.isfinite(got[starts[b] + i]).all()
    assert len(clean) < len(q) and (clean or max(m for _, m in shapes) < 9)  # (few nodes are in all windows, and the token with them)
    check_draft(y, q, k, v, table, shapes, starts, mask, 16, h, g, d, dtype, 1 / math.sqrt(d), window, rows=set(clean[:40]))
