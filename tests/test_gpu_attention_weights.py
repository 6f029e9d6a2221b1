"""Paged attention where tokens weigh next to nothing beside others, or nothing at all: they add nothing to the answer that
their weight does not (transmuter_amd/csrc/tmh_paged.hip splits each weight into two 16-bit parts)."""

import numpy as np
import pytest

import test_gpu_serving as base
from serving_plain import HALF, TINY, to_type, values
from transmuter_amd.serving import PagedCache

pytestmark = pytest.mark.gpu

D = 64


def attend(ctx, dtype, scores, v, room, page=128):
    """One head of q = (1, 0, ...) with scale 1 over tokens with the given scores (numbers that dtype holds) and values
    [tokens, D], in a table with room for `room` tokens."""
    n, pages = len(scores), -(-room // page)
    k = np.zeros((pages * page, D))
    k[:n, 0] = scores
    full = np.zeros((pages * page, D))
    full[:n] = v
    cache = PagedCache(ctx, pages, page, 1, D, dtype)
    cache.k, cache.v = (ctx.put(to_type(a.reshape(pages, page, 1, D), dtype)) for a in (k, full))
    cache.desc.k, cache.desc.v = cache.k.ptr, cache.v.ptr
    q = np.zeros((1, D))
    q[0, 0] = 1
    table = ctx.put(np.arange(pages, dtype=np.int32)[None])
    return values(cache.attend(ctx.put(to_type(q, dtype)), table, ctx.put(np.array([n], np.int32)), scale=1.0).numpy())[0]


@pytest.mark.parametrize("dtype,behind,large", [("f16", 40, 10.0), ("f16", 40, 60000.0), ("f16", 60, 60000.0), ("bf16", 300, 1e37),
                                                ("f32", 300, 1e37), ("bf16", 60, 1e4), ("f32", 60, 1e4)])
@pytest.mark.parametrize("tokens,room", [(131072, 131072), (1000, 1024), (100, 128), (100, 200000)])
def test_many_tokens_far_behind_one(ctx, dtype, behind, large, tokens, room):
    """All tokens but one lie `behind` nats below it, with large values where it has zeros and ones."""
    base.say("far behind", dtype, behind, large, tokens, room)
    scores = np.zeros(tokens)
    scores[tokens // 3] = behind
    v = np.full((tokens, D), values(to_type([large], dtype))[0])
    v[tokens // 3] = np.arange(D) % 2
    p = np.exp(scores - behind)
    want = p @ v / p.sum()
    # Each weight is rounded relatively by at most 2^-15 or, where f16 ends, by half of 2^-39 of the largest (weights below
    # that vanish: their sum is `want` itself at most); its exponential by 2^-20; then the answer's rounding.
    lost = np.minimum(want, (tokens - 1) * 2.0 ** -40 * large) if dtype == "f16" else 0
    tol = HALF[dtype] * np.abs(want) + 2.0 ** -14 * np.abs(want) + 4 * TINY[dtype] + lost
    got = attend(ctx, dtype, scores, v, room)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want).max(), tol.max())


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("tokens,room", [(5000, 5120), (1000, 1024), (100, 128), (100, 200000)])
def test_tokens_without_weight(ctx, dtype, tokens, room):
    """Scores of -infinity beside one of 0: the answer is that token's value, however large the others' are."""
    base.say("without weight", dtype, tokens, room)
    scores = np.full(tokens, -np.inf)
    scores[tokens // 2] = 0
    v = np.full((tokens, D), {"f32": 1e38, "bf16": 1e38, "f16": 65504.0}[dtype])
    v[tokens // 2] = values(to_type(np.linspace(-2, 2, D), dtype))
    got = attend(ctx, dtype, scores, v, room)
    want = v[tokens // 2]
    assert (np.abs(got - want) <= HALF[dtype] * np.abs(want) + 2.0 ** -15 * np.abs(want)).all()


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("behind", [0, 1, 5, 10, 15, 20, 24, 26])
def test_infinite_values_of_small_weight(ctx, dtype, behind):
    """An infinity at a token that weighs 2^-38 of the largest or more stays what it is; so does the rest of the row."""
    base.say("small infinities", dtype, behind)
    rng = np.random.default_rng(behind)
    scores = np.zeros(300)
    scores[7::11] = -behind - rng.integers(0, 2, len(scores[7::11])) / 64 * (behind < 26)
    v = values(to_type(rng.standard_normal((300, D)), dtype))
    for i, t in enumerate(range(7, 300, 11)):
        v[t, i] = np.inf if i % 2 else -np.inf
    many = len(range(7, 300, 11))
    got = attend(ctx, dtype, scores, v, 300)
    assert (got[:many] == np.where(np.arange(many) % 2, np.inf, -np.inf)).all()
    assert np.isfinite(got[many:]).all()


@pytest.mark.parametrize("dtype", base.TYPES)
def test_infinite_value_without_weight(ctx, dtype):
    """0 times an infinity is NaN, in its dimension only."""
    base.say("infinity without weight", dtype)
    scores = np.zeros(300)
    scores[9] = -np.inf
    v = values(to_type(np.random.default_rng(1).standard_normal((300, D)), dtype))
    v[9, 5] = np.inf
    got = attend(ctx, dtype, scores, v, 300)
    assert np.isnan(got[5]) and np.isfinite(np.delete(got, 5)).all()


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("tokens,room", [(100, 128), (200, 256), (900, 1024), (5000, 8192), (300, 200000), (100, 200000)])
def test_nothing_but_scores_of_minus_infinity(ctx, dtype, tokens, room):
    """A row whose every score is -infinity answers zeros in each way that its work is shared out, infinities and NaN among
    its values too."""
    base.say("minus infinity", dtype, tokens, room)
    v = values(to_type(np.random.default_rng(tokens).standard_normal((tokens, D)), dtype))
    v[3, 5], v[tokens // 2, 7], v[-1, 9] = np.inf, -np.inf, np.nan
    assert not attend(ctx, dtype, np.full(tokens, -np.inf), v, room).any()
