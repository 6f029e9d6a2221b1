"""The 8-bit product and paged attention against 64-bit ones in the 2-norm (serving_norms.py), at sizes that reach each of the
product's kernels, whole and in parts of K, and each way of sharing attention out (test_fp8_plan.py and
test_attention_plan.py check that they do)."""

import math

import numpy as np
import pytest

import serving_norms as norms
import test_gpu_serving as base
from serving_plain import f8_values, to_type, values
from test_gpu_attention_ways import wide_table
from transmuter_amd import serving
from transmuter_amd.serving import Fp8Weight, Rows8

pytestmark = pytest.mark.gpu

PRODUCTS = [(1, 2048, 300), (16, 4112, 530), (17, 1488, 43), (18, 1440, 2091), (17, 1632, 4149), (130, 256, 1100), (4107, 400, 5),
            (36, 1533, 8630), (17, 1472, 17464), (66, 1415, 16887), (140, 1424, 22687), (133, 3549, 23827),  # tiles, whole
            (689, 10672, 65), (49, 3487, 4193), (67, 10212, 2907), (68, 8128, 4240),                          # in parts
            (76, 1505, 24767), (199, 1514, 24890), (33, 1972, 8975), (66, 6085, 3280), (65, 6023, 6669), (512, 2048, 2048)]


@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_matmul_fp8(ctx, m, k, n):
    base.say("product in the 2-norm", m, k, n)
    rng = np.random.default_rng(m + 3 * k + n)
    a, sa = base.fp8_rows(rng, m, k)
    w, sw = base.fp8_weight(rng, n, k)
    want, spread = norms.product(f8_values(a), values(sa), f8_values(w), values(sw))
    rows, weight = Rows8(ctx.put(a, "f8_e4m3fn"), ctx.put(sa)), Fp8Weight.prepare(ctx, w, sw)
    for dtype in ("f32", "f16", "bf16"):
        y = values(serving.matmul_fp8(rows, weight, y_type=dtype).numpy())
        off, bound = norms.norm(y - want), norms.product_bound(want, spread, k, dtype)
        base.say(dtype, off / norms.norm(want), bound / norms.norm(want))
        assert off <= bound
        # ... and no row or column of it is off by itself.
        assert (np.linalg.norm(y - want, axis=1) <= 4 * bound / math.sqrt(m) + np.linalg.norm(want, axis=1) * 2 * base.HALF[dtype]).all()


ATTENTIONS = {  # lengths, tokens that the table has room for, heads, kv heads, dim, page, window
    "one sequence": ([700], 704, 16, 4, 128, 16, 0),
    "many units": ([1889, 1024], 2000, 6, 2, 256, 20, 0),
    "one unit each": ([60, 50, 33] * 40, 60, 16, 4, 64, 20, 0),
    "one unit of wide heads": ([45, 33] * 20, 60, 16, 4, 256, 20, 0),
    "half the chip": ([700, 129, 511, 1000, 300, 64] * 5, 1024, 16, 4, 128, 16, 0),
    "a window": ([5000, 2500], 8192, 8, 8, 128, 16, 1500),
    "meet": ([4000, 900], 4096, 8, 8, 128, 16, 0),
    "meet, wide heads": ([1500, 900, 1300] * 4, 2048, 8, 8, 256, 16, 0),
    "join, one head of many": ([6000], 16384, 16, 1, 128, 16, 0),
    "join, wide heads": ([3000, 40], 8192, 16, 1, 256, 32, 0),
    "long": ([9000], 9008, 32, 4, 128, 16, 0),
}


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("name", ATTENTIONS)
def test_paged_attention(ctx, name, dtype):
    base.say("attention in the 2-norm", name, dtype)
    lengths, tokens, h, g, d, page, window = ATTENTIONS[name]
    rng = np.random.default_rng(len(name) + d)
    cache, k, v, table, q = base.attention_inputs(ctx, rng, lengths, h, g, d, page, "token", dtype)
    tt = ctx.put(wide_table(rng, table, tokens, page))
    y = values(cache.attend(ctx.put(q), tt, ctx.put(np.asarray(lengths, np.int32)), window=window).numpy())
    off = bound = size = 0.0
    for i, n in enumerate(lengths):
        at = np.arange(max(0, n - window) if window else 0, n)
        where = (table[i, at // page], at % page)
        want, *rest = norms.attention(values(q[i:i + 1]).reshape(h, d), k[where], v[where], 1 / math.sqrt(d))
        b = norms.attention_bound(want, *rest, len(at), dtype)
        o = norms.norm(y[i].reshape(h, d) - want)
        assert o <= b, (i, n, o / norms.norm(want), b / norms.norm(want))
        off, bound, size = math.hypot(off, o), math.hypot(bound, b), math.hypot(size, norms.norm(want))
    base.say(off / size, bound / size)
