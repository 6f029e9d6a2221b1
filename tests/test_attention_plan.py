"""The way that paged attention's work is shared out (attention_plan in transmuter_amd/csrc/tmh_paged_plan.h) on the host:
workgroups within what HIP takes, each way where its kernel can go, and the ways that the GPU tests' cases reach."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import test_gpu_attention_each as each
import test_gpu_attention_ways as ways
import test_gpu_serving_norms as norms
from transmuter_amd import _lib
from transmuter_amd._lib import PagedCacheDesc, lib

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transmuter_amd", "csrc")
CUS = 256
JOIN, PARTS, WHOLE, WHOLE8, EACH = range(5)

# (test code only: what it compiles is the header that the kernels include)
SOURCE = r"""
#include "tmh_paged_plan.h"
extern "C" void plan(int64_t B, int64_t kv_heads, int64_t group, int head_dim, int64_t most, int64_t window, int f32, int cus, int64_t* out) {
  const tmh::AttentionPlan p = tmh::attention_plan(B, kv_heads, group, head_dim, most, window, f32 != 0, cus);
  out[0] = p.way; out[1] = p.workers; out[2] = p.units;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    path = tmp_path_factory.mktemp("plan")
    (path / "plan.cpp").write_text(SOURCE)
    subprocess.run([compiler, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", "-o",
                    str(path / "plan.so"), str(path / "plan.cpp")], check=True)
    f = ctypes.CDLL(str(path / "plan.so")).plan
    f.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] + [ctypes.c_int64] * 2 + [ctypes.c_int] * 2 + [ctypes.c_void_p]

    def call(b, kv_heads, group, dim, most, window, f32):
        out = np.zeros(3, np.int64)
        f(b, kv_heads, group, dim, most, window, int(f32), CUS, out.ctypes.data)
        return tuple(int(v) for v in out)

    return call


def check(got, b, kv_heads, group, dim, most, window, f32):
    way, workers, units = got
    unit, chunks = (64 if f32 else 128), -(-group // 16)
    items = b * kv_heads * chunks
    threads = 512 if way == WHOLE8 else 256
    assert 1 <= workers and workers * threads < 2 ** 32
    tokens = min(most, window) if window else most
    assert units == -(-tokens // unit) + (tokens < most)
    if way in (WHOLE, WHOLE8):
        assert workers == items and (way == WHOLE or dim <= 128)  # (the eight wavefronts' registers)
    elif way == EACH:
        assert workers == items * units <= CUS and tokens == most
    else:
        assert workers <= 2 * CUS  # places for parts, counters
    # Places of parts (two a worker) and counters: what the context and the workspace have.
    if way in (JOIN, EACH):
        assert workers <= 2 * CUS


@pytest.mark.parametrize("f32", [False, True])
def test_plans(plan, f32):
    rng = np.random.default_rng(int(f32))
    seen = set()
    sizes = [(int(b), int(g), int(q), int(d), int(m), int(w)) for b, g, q, d, m, w in zip(
        2 ** rng.uniform(0, 16, 20000) - .5, 2 ** rng.uniform(0, 6, 20000), 2 ** rng.uniform(0, 6, 20000),
        8 * rng.integers(1, 33, 20000), 2 ** rng.uniform(0, 18, 20000), rng.choice([0, 0, 0, 1, 100, 300, 4096], 20000))]
    # Items of one unit at and past the number of workgroups that HIP takes; no table at all.
    sizes += [(65535, 256, 1, 8, 60, 0), (65535, 257, 1, 8, 60, 0), (65535, 2 ** 15 - 1, 1, 8, 60, 0), (8, 2 ** 20, 1, 8, 60, 0),
              (65535, 16, 17, 8, 10, 0), (1, 1, 1, 64, 0, 0), (300, 4, 4, 128, 0, 0), (65535, 2 ** 20, 1, 8, 0, 0)]
    for b, g, q, d, m, w in sizes:
        b = max(b, 1)
        unit = 64 if f32 else 128
        if -(-m // unit) * b * g * -(-q // 16) >= 2 ** 31:
            continue  # (refused)
        got = plan(b, g, q, d, m, w, f32)
        check(got, b, g, q, d, m, w, f32)
        seen.add(got[0])
    assert seen == {JOIN, PARTS, WHOLE, WHOLE8, EACH}


def test_gpu_cases(plan):
    """The GPU tests' cases reach each way in each type, for heads in one block of dimensions and in more."""
    seen = set()
    for cases in (ways.CASES, each.CASES, norms.ATTENTIONS):
        for lengths, tokens, h, g, d, page, window in cases.values():
            for f32 in (False, True):
                seen.add((f32, d > 128, plan(len(lengths), g, h // g, d, -(-tokens // page) * page, window, f32)[0]))
    assert seen == {(f32, wide, way) for f32 in (False, True) for wide in (False, True) for way in range(5) if not (wide and way == WHOLE8)}


@pytest.mark.parametrize("heads,kv_heads,needle", [(2 ** 20, 2 ** 20, b"context is NULL"), (2 ** 20, 1, b"context is NULL"),
                                                   (2 ** 20 + 1, 1, b"2^20 query heads"), (2 ** 30, 2 ** 30, b"2^20 query heads")])
def test_heads(heads, kv_heads, needle):
    cache = PagedCacheDesc(k=4096, v=4096, dtype=_lib.F16, kv_heads=kv_heads, head_dim=8, page_size=16, pages=8, page_stride=2 ** 34,
                           token_stride=2 ** 30, head_stride=8)
    status = lib().tmh_paged_attention(None, 4096, heads * 8, 2, heads, ctypes.byref(cache), 4096, 4, 4096, 0.125, 0, 4096, heads * 8, None)
    assert status == (_lib.ERR_INVALID if needle == b"context is NULL" else _lib.ERR_UNSUPPORTED)
    assert needle in lib().tmh_last_error(None)
