"""The whole-number half of the paged cache (transmuter_amd/csrc/tmh_paged_plan.h) on the host: divisions, page
lookups with bad pages, spans, and that the workers' shares of ragged batches cover every unit once and leave
every part where the join looks for it."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transmuter_amd", "csrc")

# (test code only: what it compiles is the header that the kernels include)
SOURCE = r"""
#include "tmh_paged_plan.h"
using namespace tmh;
extern "C" {
uint32_t fast_div(uint32_t n, uint32_t d) { return FastDiv(d).div(n); }
int64_t offset(int64_t pages, int64_t page_size, int64_t page_stride, int64_t token_stride, const int32_t* table, uint32_t t) {
  return token_offset(PageShape{pages, page_stride, token_stride, FastDiv((uint32_t)page_size)}, table, t);
}
void span(int32_t length, int64_t most, int64_t window, int ut, int* out) {
  const Span s = span_of(length, most, window, ut);
  out[0] = s.begin; out[1] = s.end; out[2] = s.unit; out[3] = s.units;
}
uint32_t per_worker(uint32_t all, uint32_t workers) { return units_per_worker(all, workers); }
uint32_t place(uint32_t worker, int first) { return part_place(worker, first != 0); }
uint32_t parts(uint32_t first, uint32_t units, uint32_t per, uint32_t* places, uint32_t* from) {
  const Parts p = parts_of(first, units, per);
  *from = p.from;
  for (uint32_t i = 0; i < p.count; ++i) places[i] = place_of(p, i);
  return p.count;
}
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
    lib = ctypes.CDLL(str(path / "plan.so"))
    lib.fast_div.argtypes, lib.fast_div.restype = [ctypes.c_uint32] * 2, ctypes.c_uint32
    lib.offset.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_void_p, ctypes.c_uint32]
    lib.offset.restype = ctypes.c_int64
    lib.span.argtypes = [ctypes.c_int32, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_void_p]
    for f in (lib.per_worker, lib.place, lib.parts):
        f.restype = ctypes.c_uint32
    lib.parts.argtypes = [ctypes.c_uint32] * 3 + [ctypes.c_void_p] * 2
    return lib


@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 8, 10, 16, 20, 43, 86, 127, 128, 129, 255, 641, 65535, 65536, 65537,
                               2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1])
def test_division(plan, d):
    rng = np.random.default_rng(d)
    top = 2 ** 31 - 1
    ns = {0, 1, top, top - 1, d - 1, d, min(d + 1, top), top // d * d, max(top // d * d - 1, 0)}
    ns |= {int(k * d + e) for k in rng.integers(0, top // d + 1, 500) for e in (-1, 0, 1) if 0 <= k * d + e <= top}
    ns |= set(rng.integers(0, 2 ** 31, 2000).tolist())
    for n in ns:
        assert plan.fast_div(n, d) == n // d, (n, d)


def test_bad_pages_have_no_tokens(plan):
    table = np.array([3, -1, 4, 5, -2 ** 31, 2 ** 31 - 1, 0], dtype=np.int32)
    for size in (1, 16, 20):
        for t in range(len(table) * size):
            got = plan.offset(5, size, 1 << 33, 1 << 20, table.ctypes.data, t)
            page = int(table[t // size])
            assert got == ((page << 33) + (t % size << 20) if 0 <= page < 5 else -1)


@pytest.mark.parametrize("ut", [64, 128])
@pytest.mark.parametrize("window", [0, 1, 63, 64, 100, 128, 129, 1000, 2 ** 40])
def test_spans(plan, ut, window):
    out = np.zeros(4, np.int32)
    for most in (0, 1, 130, 2048, 2 ** 31 - 1):
        for length in (-2 ** 31, -1, 0, 1, 63, 64, 65, 127, 128, 129, 130, 131, 1000, 2047, 2 ** 31 - 1):
            plan.span(length, most, window, ut, out.ctypes.data)
            begin, end, unit, units = map(int, out)
            assert end == min(max(length, 0), most)
            assert begin == (max(0, end - window) if window else 0)
            if end == 0:
                assert units == 0
            else:  # the first and the last unit hold tokens of the span
                assert unit * ut <= begin < (unit + 1) * ut
                assert (unit + units - 1) * ut < end <= (unit + units) * ut


@pytest.mark.parametrize("seed", range(60))
def test_workers_cover_ragged_batches(plan, seed):
    rng = np.random.default_rng(seed)
    items = int(rng.choice([1, 2, 4, 8, 24]))
    batch = int(rng.choice([1, 2, 7, 40]))
    units = rng.integers(0, int(rng.choice([2, 4, 30, 400])) + 1, batch)
    if seed % 3 == 0:
        units[rng.random(batch) < 0.5] = 0
    workers = int(rng.choice([1, 3, 64, 512]))
    total = int(units.sum()) * items
    per = plan.per_worker(total, workers)
    if total == 0:
        assert per == 0
        return
    # What the workers do: walk their runs, an item (or a part of one) at a time.
    starts = []
    at = 0
    for b in range(batch):
        for _ in range(items):
            if units[b]:
                starts.append((at, int(units[b])))
            at += int(units[b])
    done = np.zeros(total, int)
    kept = {}  # item's first unit -> its parts' places in unit order
    used = set()
    for w in range(workers):
        at, run = w * per, w * per
        stop = min(at + per, total)
        while at < stop:
            first, n = next(s for s in starts if s[0] <= at < s[0] + s[1])
            to = min(stop, first + n)
            done[at:to] += 1
            if not (at == first and to == first + n):
                place = plan.place(w, int(at == run))
                assert place not in used and place < 2 * workers
                used.add(place)
                kept.setdefault(first, []).append(place)
            at = to
    assert (done == 1).all()
    # What the join reads.
    places = np.zeros(2 * workers + 2, np.uint32)
    source = np.zeros(1, np.uint32)
    for first, n in starts:
        count = plan.parts(first, n, per, places.ctypes.data, source.ctypes.data)
        if count == 1:
            assert first not in kept
        else:
            assert kept[first] == places[:count].tolist()
