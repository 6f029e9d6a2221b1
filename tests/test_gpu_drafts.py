"""The operators of a drafted step on the GPU against plain 64-bit implementations (drafts_plain.py): the append with head
norms, attention of trees and chains of new tokens over a paged cache, and sampling.

Tolerances are sums of half steps, as for the decoder-layer operators (test_gpu_serving.py)."""

import ctypes
import math
import sys

import numpy as np
import pytest

import drafts_plain as drafts
import serving_plain as plain
from serving_plain import HALF, TINY, to_type, values
from test_gpu_serving import APPENDS, attention_inputs, by_token, filled_cache, fp8_weight
from transmuter_amd import _lib, serving
from transmuter_amd._lib import TmhArgumentError, lib
from transmuter_amd.serving import Fp8Weight, Rows8

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
TYPES = ["f32", "f16", "bf16"]


def say(*a):
    print(*a, flush=True)


# ---------------------------------------------------------------- append with norms

# A head's squares: sixteen in a row, five levels of lanes (half steps each), the mean, eps, root, reciprocal, and the products with
# the factor, the root and gamma.
NORM = (16 + 5 + 10) * E32


def appended(x, positions, cos, sin, inter, gammas, eps, h):
    """Queries and keys [T, heads, dim] normed and turned, and the magnitudes that their rotation adds."""
    y = x.copy()
    for part, gamma in ((slice(0, h), gammas[0]), (slice(h, None), gammas[1])):
        if gamma is not None:
            y[:, part] = drafts.head_norm(y[:, part], values(gamma), eps)
    mag = np.abs(y)
    if cos is not None:
        at = np.clip(positions, 0, len(cos) - 1)
        turned = plain.rotate(y, values(cos)[at], values(sin)[at], inter)
        # |a c| + |b s| for both of a pair: the rotation of magnitudes by (|c|, -|s|) and by (|c|, |s|).
        high = plain.rotate(mag, np.abs(values(cos))[at], -np.abs(values(sin))[at], inter)
        low = plain.rotate(mag, np.abs(values(cos))[at], np.abs(values(sin))[at], inter)
        return turned, np.maximum(np.abs(high), np.abs(low))
    return y, mag


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", APPENDS, ids=str)
@pytest.mark.parametrize("which,gamma_type", [("qk", None), ("qk", "f32"), ("q", None), ("k", "bf16")])
def test_append_norm(ctx, case, dtype, which, gamma_type):
    t, h, g, d, rot, inter, page, order = case
    say("append norm", case, dtype, which, gamma_type)
    rng = np.random.default_rng(t + d + rot)
    pages = -(-2 * t // page) + 2
    cache, k0, v0 = filled_cache(ctx, rng, pages, page, g, d, dtype, order)
    qkv = to_type(rng.standard_normal((t, h + 2 * g, d)) * 2.0 ** rng.integers(-6, 6, (t, h + 2 * g, 1)), dtype).reshape(t, -1)
    slots = rng.permutation(pages * page)[:t].astype(np.int64)
    slots[rng.random(t) < 0.2] = rng.choice([-1, -2 ** 40, pages * page, 2 ** 40])
    positions = rng.integers(-3, 53, t).astype(np.int64)  # the table has 50: the ends clamp
    angle = rng.random((50, rot // 2)) * 7
    cos, sin = (to_type(np.cos(angle), "f32"), to_type(np.sin(angle), "f32")) if rot else (None, None)
    gammas = [to_type(rng.random(d) + 0.5, gamma_type or dtype) if n in which else None for n in "qk"]
    args = (ctx.put(positions), ctx.put(cos), ctx.put(sin)) if rot else ()
    norms = [ctx.put(x) if x is not None else None for x in gammas]
    eps = 1e-5
    q = cache.append(ctx.put(qkv), h, ctx.put(slots), *args, interleaved=inter, q_norm=norms[0], k_norm=norms[1], eps=eps)
    x = values(qkv).reshape(t, h + 2 * g, d)
    want, mag = appended(x[:, :h + g], positions, cos, sin, inter, gammas, eps, h)
    tol = HALF[dtype] * np.abs(want) + (NORM + 3 * E32) * mag + TINY[dtype]
    if h:
        assert (np.abs(values(q.numpy()).reshape(t, h, d) - want[:, :h]) <= tol[:, :h]).all()
    k1, v1 = cache.k.numpy(), cache.v.numpy()
    kept = (slots >= 0) & (slots < pages * page)
    at = (slots[kept] // page, slots[kept] % page)
    assert (np.abs(values(by_token(k1, order)[at]) - want[kept, h:]) <= tol[kept, h:]).all()
    assert np.array_equal(values(by_token(v1, order)[at]), x[kept, h + g:])
    # No other slot has changed.
    by_token(k1, order)[at] = by_token(k0, order)[at]
    by_token(v1, order)[at] = by_token(v0, order)[at]
    assert np.array_equal(np.asarray(k1), np.asarray(k0)) and np.array_equal(np.asarray(v1), np.asarray(v0))


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shift", [1, 3])
def test_append_norm_unaligned(ctx, inter, shift):
    """q, k, v, their gammas and tables at odd addresses and pitches, into a cache with strides of its own."""
    say("append norm unaligned", inter, shift)
    rng = np.random.default_rng(5 + shift)
    t, h, g, d, page, pages = 6, 3, 2, 24, 4, 5
    lds = {"q": h * d + 1, "k": g * d + 3, "v": g * d + 5}
    host = {n: to_type(rng.standard_normal(shift + t * ld), "f16") for n, ld in lds.items()}
    dev = {n: ctx.put(v) for n, v in host.items()}
    off = lambda t, size: ctypes.c_void_p(t.ptr.value + shift * size)  # noqa: E731
    row = {n: values(host[n])[shift:].reshape(t, lds[n])[:, :w * d].reshape(t, w, d) for n, w in (("q", h), ("k", g), ("v", g))}
    pool = np.zeros((pages, page, 64 + g * 32), np.float16)
    kt, vt = ctx.put(pool), ctx.put(pool)
    desc = _lib.PagedCacheDesc(k=kt.ptr.value + 128, v=vt.ptr.value + 128, dtype=_lib.F16, kv_heads=g, head_dim=d, page_size=page,
                               pages=pages, page_stride=page * 128, token_stride=128, head_stride=32)
    slots = np.array([3, 19, 0, -1, 8, 7], np.int64)
    positions = np.arange(t, dtype=np.int64)
    angle = rng.random((8, 12)) * 3
    tables = [np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)]
    table_dev = [ctx.put(np.concatenate([np.zeros(shift, np.float32), a.reshape(-1)])) for a in tables]
    gammas = [to_type(rng.random(d) + 0.5, "f32") for _ in "qk"]
    gamma_dev = [ctx.put(np.concatenate([np.zeros(shift, np.float32), a])) for a in gammas]
    qo = ctx.put(np.full(t * (h * d + 2), 9, np.float16))
    st, pt = ctx.put(slots), ctx.put(positions)
    ctx.check(lib().tmh_paged_append_norm(
        ctx.handle, off(dev["q"], 2), lds["q"], off(dev["k"], 2), lds["k"], off(dev["v"], 2), lds["v"], t, h, off(gamma_dev[0], 4),
        off(gamma_dev[1], 4), _lib.F32, 1e-6, pt.ptr, off(table_dev[0], 4), off(table_dev[1], 4), _lib.F32, 8, 24, int(inter),
        st.ptr, ctypes.byref(desc), qo.ptr, h * d + 2, None))
    x = np.concatenate([row["q"], row["k"]], 1)
    want, mag = appended(x, positions, *tables, inter, gammas, 1e-6, h)
    tol = HALF["f16"] * np.abs(want) + (NORM + 3 * E32) * mag + TINY["f16"]
    got = qo.numpy().reshape(t, h * d + 2)
    assert (np.abs(values(got[:, :h * d]).reshape(t, h, d) - want[:, :h]) <= tol[:, :h]).all()
    assert (got[:, h * d:] == 9).all()
    kh, vh = values(kt.numpy()), values(vt.numpy())
    wpool, vpool, tpool = np.zeros(pool.shape), np.zeros(pool.shape), np.zeros(pool.shape)
    for i, slot in enumerate(slots):
        if slot >= 0:
            for j in range(g):
                at = (slot // page, slot % page, slice(64 + 32 * j, 64 + 32 * j + d))
                wpool[at], tpool[at], vpool[at] = want[i, h + j], tol[i, h + j], row["v"][i, j]
    assert (np.abs(kh - wpool) <= tpool).all() and np.array_equal(vh, vpool)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("eps", [0.0, 1e-44, 1e-28, 1e-6])
def test_append_norm_of_any_size(ctx, dtype, eps):
    """Heads whose squares pass the largest number or fall below the smallest, and heads of zeros; an infinity and a NaN stay
    in their heads."""
    say("append norm range", dtype, eps)
    rng = np.random.default_rng(2)
    exponents = [-140, -126, -110, -76, -64, -50, -10, 0, 20, 50, 62, 65, 90, 110, 125]
    d = 64
    x = np.stack([(rng.random((3, d)) + 0.5) * rng.choice([-1, 1], (3, d)) * 2.0 ** e for e in exponents] + [np.zeros((3, d))] * 3)
    x[-2, 0, 5], x[-1, 1, 7] = np.inf, np.nan
    t = len(x)
    cache, _, _ = filled_cache(ctx, rng, 4, 16, 1, d, dtype, "token")
    gamma = to_type(np.ones(d), dtype)
    eps = float(np.float32(eps))
    q = cache.append(ctx.put(to_type(x, dtype).reshape(t, -1)), 1, ctx.put(np.arange(t)), q_norm=ctx.put(gamma), k_norm=ctx.put(gamma), eps=eps)
    got = np.stack([values(q.numpy()), values(cache.k.numpy()).reshape(-1, d)[:t]], 1)
    x = values(to_type(x, dtype))[:, :2]
    with np.errstate(invalid="ignore", over="ignore"):
        want = drafts.head_norm(x, 1.0, eps)
    for i in range(t - 2):
        for j in (0, 1):
            if eps == 0 and not x[i, j].any():
                assert np.isnan(got[i, j]).all()
            else:
                assert (np.abs(got[i, j] - want[i, j]) <= (HALF[dtype] + NORM) * np.abs(want[i, j]) + TINY[dtype] + TINY["f32"]).all(), i
    assert np.isnan(got[-2, 0, 5]) and not got[-2, 0, :5].any() and np.isnan(got[-1, 1]).all()
    if eps:
        assert not got[-2, 1].any() and not got[-1, 0].any()


# ---------------------------------------------------------------- attention of trees and chains


def draft_inputs(ctx, rng, shapes, h, g, d, page, order, dtype, kind, words=None, behind=0):
    """A cache for shapes (length, nodes), queries (with `behind` rows more), starts and masks."""
    lengths = [max(0, n) for n, _ in shapes]
    cache, k, v, table, _ = attention_inputs(ctx, rng, lengths, h, g, d, page, order, dtype)
    nodes = [n for _, n in shapes]
    starts = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    q = to_type(rng.standard_normal((starts[-1] + behind, h * d)), dtype)
    mask = None
    if kind != "chain":
        words = words or max(1, -(-max(nodes + [1]) // 64))
        mask = np.concatenate([drafts.random_tree(rng, n, words, whole=kind == "tree") for n in nodes] +
                              [rng.integers(-2 ** 62, 2 ** 62, (behind, words))])
        mask = np.ascontiguousarray(mask.astype(np.int64))
    return cache, k, v, table, q, starts, mask


def check_draft(y, q, k, v, table, shapes, starts, mask, page, h, g, d, dtype, scale, window=0, rows=None):
    """y's rows (those of `rows`, pairs of sequence and node, if given) against the 64-bit form."""
    y = values(y)
    for b, (length, n) in enumerate(shapes):
        length = max(0, length)
        at = np.arange(length)
        ids = table[b, at // page] if length else np.zeros(0, int)
        there = (ids >= 0) & (ids < len(k))
        for i in range(n):
            if rows is not None and (b, i) not in rows:
                continue
            r = starts[b] + i
            seen = drafts.sees(None if mask is None else mask[r], i, n, length, window) & there
            where = (ids[seen], at[seen] % page)
            qi = values(q[r:r + 1]).reshape(h, d)
            want, mag = plain.attend(qi, k[where], v[where], scale)
            if seen.any():
                # As check_attention has it for one token a sequence.
                size = np.abs(scale) * np.abs(qi).sum(-1).max() * np.abs(k[where]).max()
                delta = 2 * (d + 4) * 2.0 ** -24 * size + 2.0 ** -22
                tol = mag * (4 * delta + {"f32": 0, "f16": 2.0 ** -20, "bf16": 2.0 ** -15}[dtype] + (seen.sum() / 64 + 200) * E32)
            else:
                tol = np.zeros_like(want)
            tol = tol + HALF[dtype] * np.abs(want) + TINY[dtype] * 4
            got = y[r].reshape(h, d)
            bad = ~(np.abs(got - want) <= tol)
            assert not bad.any(), (b, i, length, n, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


def attend_tree(ctx, cache, q, table, lengths, starts, mask, **kw):
    return cache.attend_tree(ctx.put(q), ctx.put(table), ctx.put(np.asarray(lengths, np.int32)), ctx.put(starts),
                             ctx.put(mask) if mask is not None else None, **kw)


TREES = [  # (length, nodes) of each sequence, heads, kv heads, dim, page, order, window
    ([(1, 1)], 1, 1, 8, 1, "token", 0), ([(0, 1)], 2, 1, 64, 16, "token", 0), ([(5, 0), (0, 0), (7, 2)], 4, 2, 128, 16, "head", 0),
    ([(700, 8)], 16, 8, 128, 16, "token", 0), ([(33, 33), (40, 8), (129, 2), (64, 64), (300, 1), (0, 3)], 8, 2, 64, 16, "token", 0),
    ([(3, 7), (2, 2), (31, 40)], 4, 1, 80, 20, "head", 0), ([(1000, 100)], 8, 8, 128, 64, "head", 0),
    ([(300, 17), (17, 17), (128, 5)], 24, 1, 96, 20, "token", 0), ([(513, 12)], 16, 1, 256, 32, "token", 0),
    ([(260, 40), (40, 3)], 6, 2, 200, 8, "head", 0), ([(40, 2)] * 70, 4, 2, 64, 16, "token", 0),
    ([(5000, 30), (3, 1), (0, 0), (1200, 9)], 8, 2, 128, 16, "token", 0), ([(200, 70), (70, 70), (64, 5)], 4, 2, 128, 16, "token", 64),
    ([(300, 130), (900, 3)], 4, 1, 64, 16, "head", 1), ([(300, 20), (2000, 65)], 8, 1, 128, 256, "token", 500),
    ([(128 * 40, 4)], 1, 1, 24, 16, "token", 0), ([(260, 200)], 32, 4, 128, 16, "token", 0), ([(90, 3)] * 5, 5, 5, 136, 8, "head", 37),
    ([(64, 33), (96, 1), (50, 9)], 33, 1, 64, 7, "token", 10)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["chain", "tree", "holes"])
@pytest.mark.parametrize("case", TREES, ids=lambda c: f"b{len(c[0])}_{max(c[0])}_h{c[1]}_g{c[2]}_d{c[3]}_p{c[4]}_{c[5]}_w{c[6]}")
def test_tree_attention(ctx, case, kind, dtype):
    shapes, h, g, d, page, order, window = case
    say("tree attention", case if len(shapes) < 20 else (len(shapes), *case[1:]), kind, dtype)
    rng = np.random.default_rng(sum(n + m for n, m in shapes) + h + d)
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, page, order, dtype, kind)
    if not len(q):
        return
    y = attend_tree(ctx, cache, q, table, [n for n, _ in shapes], starts, mask, window=window).numpy()
    check_draft(y, q, k, v, table, shapes, starts, mask, page, h, g, d, dtype, 1 / math.sqrt(d), window)


@pytest.mark.parametrize("seed", range(40))
def test_random_tree_attention(ctx, seed):
    rng = np.random.default_rng(4400 + seed)
    dtype = TYPES[seed % 3]
    d = int(rng.choice([8, 40, 64, 80, 128, 128, 192, 256]))
    g = int(rng.choice([1, 2, 4]))
    h = g * int(rng.choice([1, 2, 3, 4, 7, 8, 16, 17]))
    page, order = int(rng.choice([1, 5, 8, 16, 64])), str(rng.choice(["token", "head"]))
    most = int(rng.choice([1, 5, 40, 100]))
    shapes = [(int(n), int(m)) for n, m in zip(rng.integers(0, int(rng.choice([3, 150, 1500])) + 1, 40), rng.integers(0, most + 1, 40))]
    shapes = shapes[:int(rng.choice([1, 2, 9]))]
    window, kind = int(rng.choice([0, 0, 1, 37, 128])), str(rng.choice(["chain", "tree", "holes"]))
    say("random tree attention", seed, shapes, h, g, d, page, order, window, kind, dtype)
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, page, order, dtype, kind)
    if not len(q):
        return
    scale = float(rng.choice([1 / math.sqrt(d), 0.01, -0.1]))
    y = attend_tree(ctx, cache, q, table, [n for n, _ in shapes], starts, mask, scale=scale, window=window).numpy()
    check_draft(y, q, k, v, table, shapes, starts, mask, page, h, g, d, dtype, scale, window)


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_attention_bad_pages_and_rows_behind(ctx, dtype):
    """Pages outside the cache are holes; lengths beyond the table's room clamp; rows behind the last sequence's stay as they
    were, and masks of fewer words than nodes hide the others."""
    say("tree bad pages", dtype)
    rng = np.random.default_rng(3)
    h, g, d, page = 4, 2, 64, 16
    shapes = [(100, 5), (100, 3), (64, 70), (40, 0)]
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, page, "token", dtype, "tree", words=1, behind=4)
    table[0, 2], table[0, 6] = -1, 10 ** 6
    table[1, :] = -7
    table[2, 0] = np.int32(2 ** 31 - 1)
    out = ctx.put(to_type(np.full(q.shape, 7.0), dtype))
    for m in (mask, None):
        y = attend_tree(ctx, cache, q, table, [100, 100, 64, 40], starts, m, out=out).numpy()
        check_draft(y, q, k, v, table, shapes, starts, m, page, h, g, d, dtype, 1 / 8)
        assert not values(y)[5:8].any() and (values(y)[starts[-1]:] == 7).all()
    y = attend_tree(ctx, cache, q[:5], np.ascontiguousarray(table[:1, :4]), [2 ** 31 - 1], starts[:2], mask[:5]).numpy()
    check_draft(y, q, k, v, table[:1, :4], [(64, 5)], starts, mask, page, h, g, d, dtype, 1 / 8)
    y = attend_tree(ctx, cache, q[:5], table[:1], [-3], starts[:2], mask[:5]).numpy()
    assert not values(y).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,g,d,window", [(4, 2, 64, 0), (16, 1, 128, 0), (2, 1, 256, 0), (8, 1, 40, 5)])
def test_tree_attention_hides_infinities(ctx, dtype, h, g, d, window):
    """What a row does not see has no effect on it, infinities and NaN in keys and values of the step's other tokens too, while
    the rows that see them answer with them."""
    say("tree infinities", dtype, h, g, d, window)
    rng = np.random.default_rng(9)
    page, shapes = 16, [(200, 12), (14, 14), (45, 33)]
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, page, "token", dtype, "tree")
    kb, vb = k.copy(), v.copy()
    # Of each sequence: a NaN in node 4's keys, an infinity in node 6's values, a NaN in node 7's (which others do not see).
    for b, (length, n) in enumerate(shapes):
        for node, what in ((4, "k"), (6, "inf"), (7, "nan")):
            at = length - n + node
            where = (table[b, at // page], at % page)
            if what == "k":
                kb[where] = np.nan
            else:
                vb[where] = np.inf if what == "inf" else np.nan
    cache.k, cache.v = ctx.put(to_type(kb, dtype)), ctx.put(to_type(vb, dtype))
    cache.desc.k, cache.desc.v = cache.k.ptr, cache.v.ptr
    y = attend_tree(ctx, cache, q, table, [n for n, _ in shapes], starts, mask, window=window).numpy()
    got = values(y)
    bits = np.unpackbits(mask.astype("<i8").view(np.uint8), axis=-1, bitorder="little")
    clean = []
    for b, (length, n) in enumerate(shapes):
        for i in range(n):
            r = starts[b] + i
            seen = drafts.sees(mask[r], i, n, length, window)[length - n:]
            nan, inf = seen[4] or seen[7], seen[6]
            if nan:
                assert np.isnan(got[r]).all(), (b, i)
            elif inf:
                assert not np.isfinite(got[r]).any(), (b, i)
            else:
                clean.append((b, i))
                assert np.isfinite(got[r]).all(), (b, i, bits[r][:n])
    assert clean
    # Rows that see none of these answer as without them.
    check_draft(y, q, k, v, table, shapes, starts, mask, page, h, g, d, dtype, 1 / math.sqrt(d), window, rows=clean)


def test_tree_of_one_is_attention(ctx):
    """Steps of one token a sequence agree with tmh_paged_attention."""
    say("tree of one")
    rng = np.random.default_rng(4)
    lengths = [700, 1, 0, 90, 4000]
    for dtype in TYPES:
        cache, k, v, table, q = attention_inputs(ctx, rng, lengths, 8, 2, 128, 16, "token", dtype)
        one = values(cache.attend(ctx.put(q), ctx.put(table), ctx.put(np.asarray(lengths, np.int32))).numpy())
        tree = values(attend_tree(ctx, cache, q, table, lengths, np.arange(6, dtype=np.int32), None).numpy())
        assert (np.abs(one - tree) <= 2 * HALF[dtype] * np.abs(one) + 2.0 ** -18 * np.abs(v[np.isfinite(v)]).max()).all()


WIDE = 10 ** 6  # tokens that a table has room for: of such tables tiles of many columns are worth their while


def attend_tree_wide(ctx, cache, q, table, *args, **kw):
    table = np.pad(table, ((0, 0), (0, WIDE // cache.page_size - table.shape[1])), constant_values=-1)
    return narrow(ctx, cache, q, table, *args, **kw)


narrow = attend_tree


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["chain", "tree", "holes"])
@pytest.mark.parametrize("case", TREES, ids=lambda c: f"b{len(c[0])}_{max(c[0])}_h{c[1]}_g{c[2]}_d{c[3]}_p{c[4]}_{c[5]}_w{c[6]}")
def test_tree_attention_wide_tables(ctx, case, kind, dtype):
    shapes, h, g, d, page, order, window = case
    say("tree attention, wide table", case if len(shapes) < 20 else (len(shapes), *case[1:]), kind, dtype)
    rng = np.random.default_rng(sum(n + m for n, m in shapes) + h + d + 1)
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, page, order, dtype, kind)
    if not len(q):
        return
    y = attend_tree_wide(ctx, cache, q, table, [n for n, _ in shapes], starts, mask, window=window).numpy()
    check_draft(y, q, k, v, table, shapes, starts, mask, page, h, g, d, dtype, 1 / math.sqrt(d), window)


@pytest.mark.parametrize("seed", range(20))
def test_random_tree_attention_wide_tables(ctx, seed):
    rng = np.random.default_rng(7700 + seed)
    dtype = TYPES[1 + seed % 2]
    d, g = int(rng.choice([8, 64, 104, 128, 128, 200, 256])), int(rng.choice([1, 2, 4]))
    h = g * int(rng.choice([1, 2, 4, 7, 8, 16, 17]))
    page, order, most = int(rng.choice([1, 5, 16, 64])), str(rng.choice(["token", "head"])), int(rng.choice([5, 40, 100]))
    shapes = [(int(n), int(m)) for n, m in zip(rng.integers(0, int(rng.choice([3, 150, 3000])) + 1, 9), rng.integers(0, most + 1, 9))]
    shapes, kind = shapes[:int(rng.choice([1, 2, 9]))], str(rng.choice(["chain", "tree", "holes"]))
    say("random tree attention, wide table", seed, shapes, h, g, d, page, order, kind, dtype)
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, page, order, dtype, kind)
    if not len(q):
        return
    scale = float(rng.choice([1 / math.sqrt(d), 0.01, -0.1]))
    y = attend_tree_wide(ctx, cache, q, table, [n for n, _ in shapes], starts, mask, scale=scale).numpy()
    check_draft(y, q, k, v, table, shapes, starts, mask, page, h, g, d, dtype, scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 256])
def test_tree_attention_bad_pages_in_wide_tables(ctx, dtype, d):
    say("tree bad pages, wide table", dtype, d)
    rng = np.random.default_rng(5)
    h, g, page = 8, 2, 16
    shapes = [(100, 15), (100, 13), (164, 70), (40, 0)]
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, page, "token", dtype, "tree", words=1, behind=4)
    table[0, 2], table[0, 6] = -1, 10 ** 6
    table[1, :] = -7
    table[2, 0] = np.int32(2 ** 31 - 1)
    out = ctx.put(to_type(np.full(q.shape, 7.0), dtype))
    for m in (mask, None):
        y = attend_tree_wide(ctx, cache, q, table, [100, 100, 164, 40], starts, m, out=out).numpy()
        check_draft(y, q, k, v, table, shapes, starts, m, page, h, g, d, dtype, 1 / math.sqrt(d))
        assert not values(y)[15:28].any() and (values(y)[starts[-1]:] == 7).all()
    y = attend_tree_wide(ctx, cache, q[:15], table[:1], [-3], starts[:2], mask[:15]).numpy()
    assert not values(y).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("h,g,d", [(4, 2, 64), (16, 1, 128), (2, 1, 256), (8, 1, 40)])
def test_tree_attention_hides_infinities_in_wide_tables(ctx, dtype, h, g, d, monkeypatch):
    monkeypatch.setattr(sys.modules[__name__], "attend_tree", attend_tree_wide)
    test_tree_attention_hides_infinities(ctx, dtype, h, g, d, 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["chain", "tree"])
@pytest.mark.parametrize("b,n,h,g,d,window", [(30, 70, 8, 4, 64, 100), (30, 40, 16, 4, 128, 37), (10, 70, 8, 4, 128, 1500), (16, 36, 8, 4, 256, 1100),
                                              (8, 64, 16, 4, 128, 0)])
def test_tree_attention_many_columns(ctx, b, n, h, g, d, window, kind, dtype):
    """Steps with work enough for tiles of many columns, with windows."""
    say("many columns", b, n, h, g, d, window, kind, dtype)
    rng = np.random.default_rng(b + n + window)
    shapes = [(int(x), n) for x in rng.integers(n - 3, max(1000, 2 * window), b)]
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, 16, "token", dtype, kind)
    y = attend_tree(ctx, cache, q, table, [x for x, _ in shapes], starts, mask, window=window).numpy()
    rows = {(i, j) for i in range(b) for j in (0, 1, n // 2, n - 1)}
    check_draft(y, q, k, v, table, shapes, starts, mask, 16, h, g, d, dtype, 1 / math.sqrt(d), window, rows=rows)


LONG = [  # sequences that many workgroups share, steps of many sequences: (length, nodes), heads, kv heads, dim, page, window
    ([(60000, 4)], 2, 1, 64, 64, 0), ([(30000, 20)], 8, 1, 64, 16, 0), ([(20000, 40)], 4, 1, 128, 16, 0), ([(9000, 9)], 16, 1, 256, 32, 0),
    ([(20000, 2), (3, 3), (20000, 64)], 6, 2, 72, 20, 15000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{max(c[0])}_h{c[1]}_g{c[2]}_d{c[3]}")
def test_tree_attention_long(ctx, case, dtype):
    shapes, h, g, d, page, window = case
    say("long tree attention", case, dtype)
    rng = np.random.default_rng(d + h)
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, page, "token", dtype, "tree")
    rows = {(b, i) for b, (_, n) in enumerate(shapes) for i in (0, 1, n // 2, n - 1)}
    args = (ctx, cache, q, table, [n for n, _ in shapes], starts, mask)
    y = attend_tree(*args, window=window).numpy()
    check_draft(y, q, k, v, table, shapes, starts, mask, page, h, g, d, dtype, 1 / math.sqrt(d), window, rows=rows)
    assert np.array_equal(np.asarray(attend_tree(*args, window=window).numpy()), np.asarray(y))  # (whoever joins the parts)


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_attention_many_sequences(ctx, dtype):
    say("many sequences", dtype)
    rng = np.random.default_rng(9)
    for b, h, g, d in ((3000, 2, 1, 16), (700, 24, 1, 40)):
        shapes = [(int(n), int(m)) for n, m in zip(rng.integers(0, 30, b), rng.integers(0, 4, b))]
        cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, shapes, h, g, d, 8, "head", dtype, "tree")
        y = attend_tree(ctx, cache, q, table, [n for n, _ in shapes], starts, mask).numpy()
        check_draft(y, q, k, v, table, shapes, starts, mask, 8, h, g, d, dtype, 1 / math.sqrt(d))


@pytest.mark.parametrize("heads", [2, 12, 40])
def test_tree_attention_far_offsets(ctx, heads):
    """Pages further apart than 32 bits of elements can say, as columns of one tile and of several."""
    say("tree far offsets", heads)
    d, page, stride, n = 64, 4, 2 ** 31 + 64, 3
    rng = np.random.default_rng(1)
    blocks = {p: to_type(rng.standard_normal((2, page, 1, d)), "f16") for p in range(3)}
    half = (2 * stride + page * d) * 2
    pool = ctx.alloc(2 * half)
    try:
        for p in range(3):
            for i in range(2):
                block = np.ascontiguousarray(blocks[p][i])
                ctx.check(lib().tmh_upload(ctx.handle, ctypes.c_void_p(pool.value + i * half + p * stride * 2),
                                           block.ctypes.data_as(ctypes.c_void_p), block.nbytes))
        desc = _lib.PagedCacheDesc(k=pool.value, v=pool.value + half, dtype=_lib.F16, kv_heads=1, head_dim=d, page_size=page,
                                   pages=3, page_stride=stride, token_stride=d, head_stride=0)
        q, table = to_type(rng.standard_normal((n, heads * d)), "f16"), np.array([[2, 0, 1]], np.int32)
        starts = np.array([0, n], np.int32)
        qt, tt, lt, st = ctx.put(q), ctx.put(table), ctx.put(np.array([11], np.int32)), ctx.put(starts)
        y = ctx.empty((n, heads * d), "f16")
        ctx.check(lib().tmh_paged_tree_attention(ctx.handle, qt.ptr, heads * d, n, heads, ctypes.byref(desc), tt.ptr, 1, 3, lt.ptr, st.ptr,
                                                 None, 0, 0.125, 0, y.ptr, heads * d, None))
        k, v = (np.stack([values(blocks[p][i]) for p in range(3)]) for i in range(2))
        check_draft(y.numpy(), q, k, v, table, [(11, n)], starts, None, page, heads, 1, d, "f16", 0.125)
        # ... and written there, the keys normed.
        x, gamma = to_type(rng.standard_normal((1, 2 * d)), "f16"), to_type(rng.random(d) + 0.5, "f16")
        xt, gt, slot = ctx.put(x), ctx.put(gamma), ctx.put(np.array([9], np.int64))
        ctx.check(lib().tmh_paged_append_norm(ctx.handle, None, 0, xt.ptr, 2 * d, ctypes.c_void_p(xt.ptr.value + 2 * d), 2 * d, 1, 0, None,
                                              gt.ptr, _lib.F16, 1e-6, None, None, None, 0, 0, 0, 0, slot.ptr, ctypes.byref(desc), None, 0, None))
        back = np.empty((2, d), np.float16)
        for i in range(2):
            where = ctypes.c_void_p(pool.value + i * half + (2 * stride + d) * 2)
            ctx.check(lib().tmh_download(ctx.handle, back[i].ctypes.data_as(ctypes.c_void_p), where, back[i].nbytes))
        want = drafts.head_norm(values(x)[:, None, :d], values(gamma), 1e-6)[0, 0]
        assert np.array_equal(back[1], x[0, d:])
        assert (np.abs(values(back[0]) - want) <= (HALF["f16"] + NORM + 3 * E32) * np.abs(want) + TINY["f16"]).all()
    finally:
        ctx.synchronize()
        ctx.free(pool)


# ---------------------------------------------------------------- sampling


def logits_rows(rng, t, n, dtype, spread=2.5):
    x = rng.standard_normal((t, n)) * spread
    x[:, rng.integers(0, n, min(n, 20))] += rng.exponential(3, (t, min(n, 20)))
    return to_type(x, dtype)


def check_sample(ctx, x, u, **ways):
    put = {name: ctx.put(np.asarray(v, np.int32 if name == "top_k" else np.float32)) for name, v in ways.items() if v is not None}
    got = serving.sample(ctx.put(x), ctx.put(np.asarray(u, np.float32)), **put).numpy()
    rows = values(x)
    want = [drafts.sample(rows[i], u=float(np.float32(u[i])), **{name: (int(v[i]) if name == "top_k" else float(np.float32(v[i])))
                                                                 for name, v in ways.items() if v is not None}) for i in range(len(rows))]
    assert got.dtype == np.int64 and np.array_equal(got, want), (np.flatnonzero(got != want)[:5], got[got != want][:5], np.array(want)[got != want][:5])


SAMPLES = [(1, 1), (3, 2), (5, 63), (2, 512), (7, 513), (4, 1024), (3, 1025), (2, 5000), (64, 300), (3, 32003), (2, 151936), (1, 262145)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n", SAMPLES)
def test_sample(ctx, t, n, dtype):
    say("sample", t, n, dtype)
    rng = np.random.default_rng(t + n)
    x = logits_rows(rng, t, n, dtype)
    u = rng.random(t)
    temperature = rng.choice([0.0, 0.3, 0.7, 1.0, 3.0, 100.0], t)
    top_k = rng.choice([0, 1, 2, 20, 50, 500, 5000, n, n + 1, -1], t)
    top_p = rng.choice([0.0, 0.1, 0.5, 0.9, 0.95, 0.999, 1.0, 1.5], t)
    min_p = rng.choice([0.0, 0.001, 0.05, 0.5, 1.0, 2.0], t)
    check_sample(ctx, x, u)
    check_sample(ctx, x, u, temperature=temperature)
    check_sample(ctx, x, u, top_k=top_k)
    check_sample(ctx, x, u, temperature=temperature, top_p=top_p)
    check_sample(ctx, x, u, min_p=min_p)
    check_sample(ctx, x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n", [(5, 4095), (5, 4096), (5, 4097), (5, 8191), (5, 8192), (5, 8193), (600, 8300), (1030, 20), (2, 2 ** 20 - 1)])
def test_sample_sizes(ctx, t, n, dtype):
    """About the longest row of one workgroup, more rows than a launch takes, and the longest row."""
    say("sample sizes", t, n, dtype)
    rng = np.random.default_rng(t * n)
    x = logits_rows(rng, t, n, dtype)
    check_sample(ctx, x, rng.random(t), temperature=rng.choice([0.0, 0.5, 1.0, 4.0], t), top_k=rng.choice([0, 1, 64, 65, 900], t),
                 top_p=rng.choice([0.2, 0.9, 0.9999, 1.0], t), min_p=rng.choice([0.0, 0.01, 0.3], t))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [4, 1000, 40000])
def test_sample_equal_logits(ctx, n, dtype):
    """Whole rows of one value, and of few: the first of equals are kept, each as likely as the other."""
    say("sample equals", n, dtype)
    rng = np.random.default_rng(n)
    few = rng.integers(0, 3, (12, n)).astype(np.float64)
    for x in (np.zeros((12, n)), np.full((12, n), -3.5), few, few * 0.5 - 20):
        u = np.concatenate([[0.0, 0.5, 0.25, 1 - 2.0 ** -24, 2.0 ** -24], rng.random(7)])
        x = to_type(x, dtype)
        check_sample(ctx, x, u)
        check_sample(ctx, x, u, top_k=np.array([1, 2, 3, n // 2, n - 1, n, 0, 7, 1, 2, 3, 4]))
        check_sample(ctx, x, u, top_p=np.array([0.5, 0.25, 0.75, 0.1, 0.9, 0.99, 1.0, 0.0, 2.0 ** -24, 0.5, 0.125, 1 - 2.0 ** -24]))
        check_sample(ctx, x, u, top_k=np.full(12, n // 2 + 1), top_p=np.linspace(0.05, 1, 12))
        check_sample(ctx, x, u, min_p=np.linspace(0, 1, 12))


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_special(ctx, dtype):
    """Masked tokens, infinities, NaN, -0 beside 0; temperatures, top-p, min-p and random numbers at and past their ends."""
    say("sample special", dtype)
    n = 3000
    rng = np.random.default_rng(1)
    x = logits_rows(rng, 9, n, "f32").astype(np.float64)
    x[0] = -np.inf
    x[1, rng.permutation(n)[:n - 3]] = -np.inf
    x[2, ::2] = np.nan
    x[3, [100, 2000]] = np.inf
    x[4] = np.where(np.arange(n) % 2, 0.0, -0.0)
    x[5] = np.nan
    x[6, :] = -np.inf
    x[6, n - 1] = -60000.0
    x[7] *= 1000
    x = to_type(x, dtype)
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        us = np.full(9, u)
        check_sample(ctx, x, us)
        for temperature in (0.0, -1.0, np.nan, 1e-30, 1e30, np.inf, 0.7):
            check_sample(ctx, x, us, temperature=np.full(9, temperature))
        for k in (1, 2, 5, 2999, 3000, -5):
            check_sample(ctx, x, us, top_k=np.full(9, k))
        for p in (-1.0, 0.0, 1e-30, 0.5, np.nan, 1 - 2.0 ** -24):
            check_sample(ctx, x, us, top_p=np.full(9, p))
        for p in (-1.0, np.nan, 1e-20, 1.0, np.inf):
            check_sample(ctx, x, us, min_p=np.full(9, p))
        check_sample(ctx, x, us, temperature=np.full(9, 0.9), top_k=np.full(9, 40), top_p=np.full(9, 0.8), min_p=np.full(9, 0.1))
    check_sample(ctx, x, np.full(9, 1.0))
    check_sample(ctx, x, np.full(9, 7.0), top_k=np.full(9, 3))


@pytest.mark.parametrize("pitch,shift,dtype", [(1003, 1, "f16"), (1001, 3, "bf16"), (1001, 1, "f32"), (1008, 0, "f16")])
def test_sample_strides(ctx, pitch, shift, dtype):
    """Rows with a pitch, at any address."""
    say("sample strides", pitch, shift, dtype)
    t, n = 6, 1000
    rng = np.random.default_rng(pitch)
    x = logits_rows(rng, t, pitch, dtype)
    x[:, n:] = to_type(np.full(1, 900.0), dtype)[0]  # (what lies between the rows is not read)
    flat = np.concatenate([x.reshape(-1)[:shift], x.reshape(-1)])
    dev = ctx.put(flat) if dtype != "bf16" else ctx.put(np.ascontiguousarray(flat), "bf16")
    u = rng.random(t).astype(np.float32)
    ut, out = ctx.put(u), ctx.empty((t,), "s64")
    k, p = ctx.put(np.full(t, 30, np.int32)), ctx.put(np.full(t, 0.9, np.float32))
    at = ctypes.c_void_p(dev.ptr.value + shift * (4 if dtype == "f32" else 2))
    ctx.check(lib().tmh_sample(ctx.handle, at, pitch, dev.tmh_dtype, t, n, None, k.ptr, p.ptr, None, ut.ptr, out.ptr, None))
    rows = values(x)[:, :n]
    assert np.array_equal(out.numpy(), [drafts.sample(rows[i], top_k=30, top_p=float(np.float32(0.9)), u=float(u[i])) for i in range(t)])


def test_sample_is_as_likely_as_its_weights(ctx):
    """Many random numbers over one distribution: counts within five standard deviations of their means."""
    say("sample counts")
    rng = np.random.default_rng(0)
    row = rng.standard_normal(40) * 2
    t = 20000
    x = np.tile(row, (t, 1)).astype(np.float32)
    u = (np.arange(t) + 0.5) / t
    tokens = serving.sample(ctx.put(x), ctx.put(u.astype(np.float32)), top_k=ctx.put(np.full(t, 10, np.int32))).numpy()
    w = np.exp(values(x[0]))
    w[np.argsort(-w)[10:]] = 0
    w /= w.sum()
    # Evenly spaced random numbers: each token as often as its share, to one at either end.
    assert (np.abs(np.bincount(tokens, minlength=40) - t * w) <= 2).all()


# ---------------------------------------------------------------- a drafted step, streams and graphs


class Step:
    """A step of drafted tokens over one cache as a program runs it: append with head norms, attention, logits, tokens, and the rows of
    a path appended once more to the slots that follow each other."""

    SHAPES = [(45, 5), (708, 8), (3, 3), (0, 0), (130, 1)]  # tokens with the step's own, of those the step's
    H, G, D, PAGE, V = 4, 2, 64, 16, 9000

    def __init__(self, ctx, rng):
        h, g, d, page = self.H, self.G, self.D, self.PAGE
        self.ctx = ctx
        self.cache, _, _, self.table, _, self.starts, _ = draft_inputs(ctx, rng, self.SHAPES, h, g, d, page, "token", "f16", "chain")
        self.t = t = int(self.starts[-1])
        self.first = [n - m for n, m in self.SHAPES]
        parents = [[-1] + [int(rng.integers(0, i)) for i in range(1, m)] for _, m in self.SHAPES]
        seen, depth = np.zeros((t, 64), bool), np.zeros(t, np.int64)
        self.paths, slots, kept = [], np.zeros(t, np.int64), np.full(t, -1, np.int64)
        for b, (_, m) in enumerate(self.SHAPES):
            for i in range(m):
                r, up = self.starts[b] + i, parents[b][i]
                if up >= 0:
                    seen[r], depth[r] = seen[self.starts[b] + up], depth[self.starts[b] + up] + 1
                seen[r, i] = True
                slots[r] = self.slot(b, self.first[b] + i)
            path = np.flatnonzero(seen[self.starts[b] + m - 1]) if m else np.zeros(0, int)
            self.paths.append(self.starts[b] + path)
            for j, i in enumerate(path):
                kept[self.starts[b] + i] = self.slot(b, self.first[b] + j)
        self.mask = drafts.pack(seen)
        first = np.repeat(self.first, [m for _, m in self.SHAPES])
        angle = rng.random((800, d // 2)) * 6
        self.gammas = [to_type(rng.random(d) + 0.5, "f16") for _ in range(2)]
        put = ctx.put
        self.dev = dict(qkv=ctx.empty((t, (h + 2 * g) * d), "f16"), u=ctx.empty((t,), "f32"), positions=put(first + depth), slots=put(slots),
                        kept=put(kept), table=put(self.table), lengths=put(np.array([n for n, _ in self.SHAPES], np.int32)),
                        starts=put(self.starts), mask=put(self.mask), cos=put(np.cos(angle).astype(np.float32)),
                        sin=put(np.sin(angle).astype(np.float32)), gq=put(self.gammas[0]), gk=put(self.gammas[1]),
                        p=put(np.full(t, 0.9, np.float32)), k=put(np.where(np.arange(t) % 2, 50, 0).astype(np.int32)))
        w, sw = fp8_weight(rng, self.V, h * d)
        self.head = Fp8Weight.prepare(ctx, w, sw * np.float32(0.02))
        self.q, self.y = ctx.empty((t, h * d), "f16"), ctx.empty((t, h * d), "f16")
        self.rows, self.logits, self.tokens = Rows8.empty(ctx, (t, h * d)), ctx.empty((t, self.V), "f16"), ctx.empty((t,), "s64")

    def slot(self, b, token):
        return int(self.table[b, token // self.PAGE]) * self.PAGE + token % self.PAGE

    def fill(self, rng):
        qkv, u = to_type(rng.standard_normal((self.t, self.dev["qkv"].shape[1])), "f16"), rng.random(self.t).astype(np.float32)
        for name, v in (("qkv", qkv), ("u", u)):
            self.ctx.check(lib().tmh_upload(self.ctx.handle, self.dev[name].ptr, v.ctypes.data_as(ctypes.c_void_p), v.nbytes))
        return u

    def append(self, slots):
        v, c = self.dev, self.cache
        c.append(v["qkv"], self.H, slots, v["positions"], v["cos"], v["sin"], q_norm=v["gq"], k_norm=v["gk"], out=self.q)

    def run(self):
        v, ctx, c, w = self.dev, self.ctx, self.cache, self.H * self.D
        self.append(v["slots"])
        c.attend_tree(self.q, v["table"], v["lengths"], v["starts"], v["mask"], out=self.y)
        ctx.check(lib().tmh_quantize_rows(ctx.handle, self.y.ptr, w, None, 0, _lib.F16, self.t, w, self.rows.q.ptr, w, self.rows.scales.ptr, None))
        ctx.check(lib().tmh_matmul_fp8(ctx.handle, self.head.handle, self.rows.q.ptr, self.t, w, self.rows.scales.ptr, None, 0, self.logits.ptr,
                                       _lib.F16, self.V, None))
        serving.sample(self.logits, v["u"], top_k=v["k"], top_p=v["p"], out=self.tokens)
        self.append(v["kept"])

    def results(self):
        return [np.asarray(v.numpy()).copy() for v in (self.q, self.y, self.logits, self.tokens, self.cache.k, self.cache.v)]

    def clear(self):
        for v in (self.q, self.y, self.logits, self.tokens):
            zero = np.zeros(v.nbytes, np.uint8)
            self.ctx.check(lib().tmh_upload(self.ctx.handle, v.ptr, zero.ctypes.data_as(ctypes.c_void_p), v.nbytes))

    def graph(self):
        graph = ctypes.c_void_p()
        self.ctx.check(lib().tmh_graph_begin(self.ctx.handle, None))
        self.run()
        self.ctx.check(lib().tmh_graph_end(self.ctx.handle, None, ctypes.byref(graph)))
        return graph


def same(a, b):
    return all(np.array_equal(x, y, equal_nan=x.dtype.kind == "f") for x, y in zip(a, b))


def test_drafted_step(ctx):
    """Its answers, its tokens, and that the path that was kept answers afterwards as a chain what it did as a branch of its tree."""
    say("drafted step")
    rng = np.random.default_rng(6)
    s = Step(ctx, rng)
    u = s.fill(rng)
    s.append(s.dev["slots"])
    k, v = (values(np.asarray(x.numpy())) for x in (s.cache.k, s.cache.v))
    s.run()
    q, y, logits, tokens, k_then, v_then = s.results()
    geometry = (s.PAGE, s.H, s.G, s.D, "f16", 1 / math.sqrt(s.D))
    check_draft(y, q, k, v, s.table, s.SHAPES, s.starts, s.mask, *geometry)
    rows = values(logits)
    assert tokens.tolist() == [drafts.sample(rows[i], top_k=50 * (i % 2), top_p=float(np.float32(0.9)), u=float(u[i])) for i in range(s.t)]
    lengths = [a + len(path) for a, path in zip(s.first, s.paths)]
    starts = np.concatenate([[0], np.cumsum([len(path) for path in s.paths])]).astype(np.int32)
    chosen = q[np.concatenate(s.paths)]
    chain = s.cache.attend_tree(ctx.put(chosen), s.dev["table"], ctx.put(np.array(lengths, np.int32)), ctx.put(starts)).numpy()
    check_draft(chain, chosen, values(k_then), values(v_then), s.table, [(n, len(path)) for n, path in zip(lengths, s.paths)], starts, None, *geometry)
    # (Over the same keys and values, bit for bit, so both are within those bounds of the same numbers.)
    slots, kept = s.dev["slots"].numpy(), s.dev["kept"].numpy()
    r = np.flatnonzero(kept >= 0)
    for before, then in ((k, k_then), (v, v_then)):
        at, to = ((x[r] // s.PAGE, x[r] % s.PAGE) for x in (slots, kept))
        assert np.array_equal(before[at], values(then)[to])


def test_drafted_step_in_graphs(ctx):
    """The step recorded twice on one context, whose workspace both graphs share and larger calls between the replays let grow: every
    replay gives the eager calls' bits."""
    say("drafted step in graphs")
    rng = np.random.default_rng(7)
    steps = [Step(ctx, rng), Step(ctx, rng)]
    for s in steps:
        s.fill(rng)
        s.run()
    first = steps[0].results()
    steps[0].run()
    assert same(first, steps[0].results())
    graphs = [s.graph() for s in steps]
    for replay in range(4):
        wants = []
        for s in steps:
            s.fill(rng)
            s.run()
            wants.append(s.results())
            s.clear()
        serving.sample(ctx.put(to_type(rng.standard_normal((8 << replay, 9000)), "f32")), ctx.put(rng.random(8 << replay).astype(np.float32)),
                       top_k=ctx.put(np.full(8 << replay, 9, np.int32)))
        for graph in graphs:
            ctx.check(lib().tmh_graph_launch(ctx.handle, graph, None))
        for s, want in zip(steps, wants):
            assert same(want, s.results()), replay
        ctx.synchronize()
    for graph in graphs:
        ctx.check(lib().tmh_graph_destroy(ctx.handle, graph))


def test_drafts_on_another_stream(ctx):
    """The calls run on the stream they are given: a second context's, fenced by the host."""
    from transmuter_amd import Context

    say("drafts on another stream")
    rng = np.random.default_rng(8)
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, [(300, 9), (20, 3)], 8, 2, 64, 16, "token", "f16", "tree")
    args = ctx.put(q), ctx.put(table), ctx.put(np.array([300, 20], np.int32)), ctx.put(starts), ctx.put(mask)
    x, u = ctx.put(logits_rows(rng, 3, 9000, "f16")), ctx.put(rng.random(3).astype(np.float32))
    qkv, slots = ctx.put(to_type(rng.standard_normal((2, 12 * 64)), "f16")), ctx.put(np.array([-1, -1], np.int64))
    gamma = ctx.put(to_type(rng.random(64), "f16"))

    def calls(stream):
        return (cache.attend_tree(*args, stream=stream), serving.sample(x, u, stream=stream),
                cache.append(qkv, 8, slots, q_norm=gamma, stream=stream))

    want = [y.numpy() for y in calls(None)]
    other = Context(0)
    try:
        got = calls(other.stream)
        other.synchronize()
        assert all(np.array_equal(y.numpy(), w) for y, w in zip(got, want))
    finally:
        other.close()


def test_drafts_refused_in_a_capture():
    """A fresh context's capture finds no workspace for the attention or for long rows of logits: refused, not run. Short rows need none."""
    from transmuter_amd import Context

    say("drafts refused in a capture")
    c = Context(0)
    try:
        cache = serving.PagedCache(c, 4, 16, 1, 64)
        q, table, lengths, y = c.empty((1, 64), "f16"), c.put(np.array([[0]], np.int32)), c.put(np.array([3], np.int32)), c.empty((1, 64), "f16")
        starts, x, u, token = c.put(np.array([0, 1], np.int32)), c.put(np.zeros((1, 9000), np.float32)), c.put(np.zeros(1, np.float32)), c.empty((1,), "s64")
        x.numpy()
        c.check(lib().tmh_graph_begin(c.handle, None))
        one = lib().tmh_paged_tree_attention(c.handle, q.ptr, 64, 1, 1, ctypes.byref(cache.desc), table.ptr, 1, 1, lengths.ptr, starts.ptr, None, 0, 1.0,
                                             0, y.ptr, 64, None)
        needle = lib().tmh_last_error(c.handle)
        two = lib().tmh_sample(c.handle, x.ptr, 9000, _lib.F32, 1, 9000, None, None, None, None, u.ptr, token.ptr, None)
        needles = needle, lib().tmh_last_error(c.handle)
        three = lib().tmh_sample(c.handle, x.ptr, 4096, _lib.F32, 1, 4096, None, None, None, None, u.ptr, token.ptr, None)
        graph = ctypes.c_void_p()
        c.check(lib().tmh_graph_end(c.handle, None, ctypes.byref(graph)))
        c.check(lib().tmh_graph_launch(c.handle, graph, None))
        assert token.numpy().tolist() == [0]
        c.check(lib().tmh_graph_destroy(c.handle, graph))
        assert (one, two, three) == (_lib.ERR_UNSUPPORTED, _lib.ERR_UNSUPPORTED, 0)
        assert all(b"before the capture" in n for n in needles)
    finally:
        c.close()


# ---------------------------------------------------------------- refusals that need a device


def test_refusals(ctx):
    say("refusals")
    rng = np.random.default_rng(0)
    cache, k, v, table, q, starts, mask = draft_inputs(ctx, rng, [(20, 3)], 2, 1, 64, 16, "token", "f16", "tree")
    ok = dict(q=ctx.put(q), page_table=ctx.put(table), lengths=ctx.put(np.array([20], np.int32)), starts=ctx.put(starts), mask=ctx.put(mask))
    cache.attend_tree(**ok)
    gone = ctx.put(mask)
    gone.free()
    for kw in (dict(starts=ctx.put(starts[:1])), dict(starts=ctx.put(starts.astype(np.int64))), dict(mask=ctx.put(mask[:2])),
               dict(mask=ctx.put(mask.astype(np.int32))), dict(mask=gone), dict(lengths=ctx.put(np.zeros(2, np.int32))),
               dict(window=-1), dict(scale=math.nan), dict(q=ctx.put(q[:, :96].copy())), dict(q=ctx.put(q.astype(np.float32)))):
        with pytest.raises(TmhArgumentError):
            cache.attend_tree(**{**ok, **kw})
    x, u = ctx.put(np.zeros((2, 9), np.float32)), ctx.put(np.zeros(2, np.float32))
    for kw in (dict(random=ctx.put(np.zeros(3, np.float32))), dict(top_k=u), dict(temperature=ctx.put(np.zeros(2, np.float16))),
               dict(logits=ctx.put(np.zeros((2, 9), np.int32))), dict(out=ctx.empty((2,), "s32")), dict(top_p=gone)):
        with pytest.raises(TmhArgumentError):
            serving.sample(**{**dict(logits=x, random=u), **kw})
    qkv, slots = ctx.put(np.zeros((2, 4 * 64), np.float16)), ctx.put(np.zeros(2, np.int64))
    gamma = ctx.put(np.ones(64, np.float16))
    for kw in (dict(q_norm=ctx.put(np.ones(32, np.float16))), dict(q_norm=gamma, k_norm=ctx.put(np.ones(64, np.float32))),
               dict(q_norm=gamma, eps=-1.0), dict(q_norm=gamma, eps=math.nan), dict(k_norm=ctx.put(np.ones(64, np.int32)))):
        with pytest.raises(TmhArgumentError):
            cache.append(qkv, 2, slots, **kw)
