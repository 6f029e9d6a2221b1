"""Attention over a paged cache whose table is so narrow that every unit it has room for gets a workgroup, which asks for its
rows before it knows the sequence's length (EACH in transmuter_amd/csrc/tmh_paged.hip). Behind a sequence's own pages the
tables hold any numbers. Tolerances as in test_gpu_serving.py."""

import ctypes
import math

import numpy as np
import pytest

import test_gpu_serving as base
from test_gpu_attention_ways import wide_table
from serving_plain import to_type
from transmuter_amd._lib import lib

pytestmark = pytest.mark.gpu

CASES = {  # lengths, tokens that the table has room for, heads, kv heads, dim, page, window
    "one sequence": ([700], 704, 16, 4, 128, 16, 0),
    "one token in a table of many": ([1], 1500, 8, 2, 128, 16, 0),
    "nothing in a table of many": ([0], 1500, 8, 2, 128, 16, 0),
    "borders of units": ([0, 1, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 384, 385, 512], 512, 4, 2, 64, 16, 0),
    "full tables": ([512, 512, 511], 512, 8, 2, 128, 32, 0),
    "pages that end in a tile": ([300, 0, 77, 299], 301, 8, 4, 80, 7, 0),
    "pages of one token": ([260, 3, 0], 400, 8, 2, 96, 1, 0),
    "one page": ([300, 0, 512], 512, 8, 2, 128, 512, 0),
    "wide heads": ([200, 0, 256, 129], 256, 12, 4, 256, 16, 0),
    "wide heads of many units": ([1889, 5, 1024], 2000, 6, 2, 256, 20, 0),
    "two chunks of heads": ([300, 0, 77], 640, 20, 1, 40, 16, 0),
    "a window as long as the table": ([300, 0, 640], 640, 8, 2, 128, 16, 640),
    "as many units as compute units": ([4096, 1, 0, 2000], 4096, 4, 2, 128, 16, 0),
    "narrow heads": ([600, 1], 640, 3, 3, 8, 16, 0),
}


@pytest.mark.parametrize("order", ["token", "head"])
@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("name", CASES)
def test_each(ctx, name, dtype, order):
    base.say("each", name, dtype, order)
    lengths, tokens, h, g, d, page, window = CASES[name]
    rng = np.random.default_rng(len(name) + d)
    cache, k, v, table, q = base.attention_inputs(ctx, rng, lengths, h, g, d, page, order, dtype)
    tt, lt, qt = ctx.put(wide_table(rng, table, tokens, page)), ctx.put(np.asarray(lengths, np.int32)), ctx.put(q)
    y = cache.attend(qt, tt, lt, window=window).numpy()
    base.check_attention(y, q, k, v, table, lengths, page, h, g, d, dtype, 1 / math.sqrt(d), window)
    other = ctx.put(np.asarray([(n * 7 + 3) % 129 if n else 0 for n in lengths], np.int32))
    for i in range(6):
        if i % 2:
            cache.attend(qt, tt, other, window=window)
        assert np.array_equal(np.asarray(cache.attend(qt, tt, lt, window=window).numpy()), np.asarray(y), equal_nan=True)


@pytest.mark.parametrize("lengths", [[-1, -2 ** 31, 0], [2 ** 31 - 1, 5000, 641]])
def test_lengths_outside_the_table(ctx, lengths):
    """Lengths below zero are none, lengths past the table are the table's."""
    base.say("each, lengths", lengths)
    tokens, h, g, d, page = 640, 8, 2, 128, 16
    full = [min(max(n, 0), tokens) for n in lengths]
    rng = np.random.default_rng(3)
    cache, k, v, table, q = base.attention_inputs(ctx, rng, full, h, g, d, page, "token", "f16")
    tt, lt, qt = ctx.put(wide_table(rng, table, tokens, page)), ctx.put(np.asarray(lengths, np.int32)), ctx.put(q)
    y = cache.attend(qt, tt, lt).numpy()
    base.check_attention(y, q, k, v, table, full, page, h, g, d, "f16", 1 / math.sqrt(d), 0)


@pytest.mark.parametrize("name", ["one sequence", "borders of units", "wide heads of many units"])
def test_each_in_a_graph(ctx, name):
    """Recorded once and replayed over lengths that change between the replays, with eager calls in between."""
    base.say("each in a graph", name)
    lengths, tokens, h, g, d, page, window = CASES[name]
    rng = np.random.default_rng(5)
    cache, k, v, table, q = base.attention_inputs(ctx, rng, lengths, h, g, d, page, "token", "bf16")
    tt, lt, qt, y = ctx.put(wide_table(rng, table, tokens, page)), ctx.put(np.asarray(lengths, np.int32)), ctx.put(q), ctx.empty(q.shape, "bf16")
    cache.attend(qt, tt, lt, out=y)
    ctx.check(lib().tmh_graph_begin(ctx.handle, None))
    cache.attend(qt, tt, lt, out=y)
    graph = ctypes.c_void_p()
    ctx.check(lib().tmh_graph_end(ctx.handle, None, ctypes.byref(graph)))
    for replay in range(4):
        now = np.asarray([int(n * f) for n, f in zip(lengths, rng.random(len(lengths)))], np.int32) if replay else np.asarray(lengths, np.int32)
        ctx.check(lib().tmh_upload(ctx.handle, lt.ptr, now.ctypes.data_as(ctypes.c_void_p), now.nbytes))
        ctx.check(lib().tmh_upload(ctx.handle, y.ptr, to_type(np.full(q.shape, 9.0), "bf16").ctypes.data_as(ctypes.c_void_p), y.nbytes))
        ctx.check(lib().tmh_graph_launch(ctx.handle, graph, None))
        got = y.numpy().copy()
        assert np.array_equal(got, cache.attend(qt, tt, lt).numpy())
        base.check_attention(got, q, k, v, table, [int(n) for n in now], page, h, g, d, "bf16", 1 / math.sqrt(d), window)
    ctx.synchronize()
    ctx.check(lib().tmh_graph_destroy(ctx.handle, graph))
