"""Attention over a paged cache in each of the ways that its work is shared out (transmuter_amd/csrc/tmh_paged.hip: items
whole, parts that meet in the kernel, parts that a second kernel joins), which the width of the page table and the
number of items decide. Tolerances as in test_gpu_serving.py."""

import ctypes
import math

import numpy as np
import pytest

import test_gpu_serving as base
from serving_plain import to_type
from transmuter_amd._lib import lib

pytestmark = pytest.mark.gpu

RAGGED = [0, 1, 700, 0, 129, 511, 512, 513, 64, 1000, 2, 300, 0, 128, 256, 33]
CASES = {  # lengths, tokens that the table has room for, heads, kv heads, dim, page, window
    "whole, one short sequence": ([300], 512, 8, 2, 128, 16, 0),
    "whole, half the chip": (RAGGED * 2, 1024, 16, 4, 128, 16, 0),
    "whole, a window": ([700, 0, 5, 1024] * 8, 1024, 8, 4, 64, 32, 100),
    "whole, two chunks of heads": ([400, 0, 77], 448, 40, 2, 80, 7, 0),
    "whole, one unit": ([1, 0, 128, 77, 5] * 60, 128, 8, 2, 128, 16, 0),
    "whole, one unit of wide heads": ([1, 0, 45, 33] * 20, 60, 16, 4, 256, 20, 0),
    "whole, a window in a long table": ([5000, 0, 100, 129, 1], 8192, 8, 2, 128, 16, 100),
    "whole, a window of wide heads": ([900, 0, 70, 128], 4096, 64, 4, 256, 16, 60),
    "meet, few items": ([1, 4000, 900], 4096, 8, 8, 128, 16, 0),
    "meet, one sequence": ([2111], 2112, 16, 4, 128, 64, 0),
    "meet, many sequences": (RAGGED * 10, 2048, 4, 2, 64, 16, 0),
    "meet, one long among short": ([3] * 30 + [9000] + [0] * 5, 9216, 8, 4, 96, 16, 0),
    "meet, a window": ([5000, 100, 0, 2500], 8192, 8, 8, 128, 16, 1500),
    "meet, wide heads": ([1500, 0, 1300], 2048, 4, 4, 256, 16, 0),
    "join, one head of many": ([6000], 16384, 16, 1, 128, 16, 0),
    "join, short in a wide table": ([300, 0, 1], 60000, 32, 2, 128, 16, 0),
    "join, wide heads": ([3000, 40], 8192, 16, 1, 256, 32, 0),
}


def wide_table(rng, table, tokens, page):
    """The table with room for `tokens`: behind the sequences' own pages any numbers."""
    width = -(-tokens // page)
    assert width >= table.shape[1]
    out = rng.integers(-2 ** 31, 2 ** 31, (len(table), width)).astype(np.int32)
    out[:, :table.shape[1]] = table
    return out


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("name", CASES)
def test_ways(ctx, name, dtype):
    base.say("way", name, dtype)
    lengths, tokens, h, g, d, page, window = CASES[name]
    rng = np.random.default_rng(len(name) + d)
    cache, k, v, table, q = base.attention_inputs(ctx, rng, lengths, h, g, d, page, "token", dtype)
    tt, lt, qt = ctx.put(wide_table(rng, table, tokens, page)), ctx.put(np.asarray(lengths, np.int32)), ctx.put(q)
    y = cache.attend(qt, tt, lt, window=window).numpy()
    base.check_attention(y, q, k, v, table, lengths, page, h, g, d, dtype, 1 / math.sqrt(d), window)
    # The same bits again, whoever comes last where parts meet, and after calls that left their own parts behind.
    other = ctx.put(np.asarray([(n * 7 + 3) % 129 if n else 0 for n in lengths], np.int32))
    for i in range(6):
        if i % 2:
            cache.attend(qt, tt, other, window=window)
        assert np.array_equal(np.asarray(cache.attend(qt, tt, lt, window=window).numpy()), np.asarray(y), equal_nan=True)


@pytest.mark.parametrize("name", ["whole, half the chip", "meet, many sequences", "meet, one sequence", "join, one head of many"])
def test_ways_in_a_graph(ctx, name):
    """Recorded once and replayed over lengths that change between the replays, with eager calls in between."""
    base.say("way in a graph", name)
    lengths, tokens, h, g, d, page, window = CASES[name]
    rng = np.random.default_rng(5)
    cache, k, v, table, q = base.attention_inputs(ctx, rng, lengths, h, g, d, page, "token", "f16")
    wide = wide_table(rng, table, tokens, page)
    tt, lt, qt, y = ctx.put(wide), ctx.put(np.asarray(lengths, np.int32)), ctx.put(q), ctx.empty(q.shape, "f16")

    def call(out):
        ctx.check(lib().tmh_paged_attention(ctx.handle, qt.ptr, h * d, len(lengths), h, ctypes.byref(cache.desc), tt.ptr, wide.shape[1],
                                            lt.ptr, 1 / math.sqrt(d), window, out.ptr, h * d, None))

    call(y)
    ctx.check(lib().tmh_graph_begin(ctx.handle, None))
    call(y)
    graph = ctypes.c_void_p()
    ctx.check(lib().tmh_graph_end(ctx.handle, None, ctypes.byref(graph)))
    eager = ctx.empty(q.shape, "f16")
    for replay in range(4):
        now = np.asarray([int(n * f) for n, f in zip(lengths, rng.random(len(lengths)))], np.int32) if replay else np.asarray(lengths, np.int32)
        ctx.check(lib().tmh_upload(ctx.handle, lt.ptr, now.ctypes.data_as(ctypes.c_void_p), now.nbytes))
        ctx.check(lib().tmh_upload(ctx.handle, y.ptr, to_type(np.full(q.shape, 9.0), "f16").ctypes.data_as(ctypes.c_void_p), y.nbytes))
        ctx.check(lib().tmh_graph_launch(ctx.handle, graph, None))
        got = y.numpy().copy()
        call(eager)
        assert np.array_equal(got, eager.numpy())
        base.check_attention(got, q, k, v, table, [int(n) for n in now], page, h, g, d, "f16", 1 / math.sqrt(d), window)
    ctx.synchronize()
    ctx.check(lib().tmh_graph_destroy(ctx.handle, graph))
