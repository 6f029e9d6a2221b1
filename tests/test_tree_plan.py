"""What the rows of a drafted step see (transmuter_amd/csrc/tmh_tree_plan.h) on the host, against a plain restatement."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import drafts_plain as drafts

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transmuter_amd", "csrc")

# (test code only: what it compiles is the header that the kernels include)
SOURCE = r"""
#include "tmh_tree_plan.h"
using namespace tmh;
extern "C" {
uint32_t bits_of(const uint64_t* words, int count, int first) { return tree_bits(words, count, first); }
uint32_t bits_of_chain(int node, int first) { return chain_bits(node, first); }
uint32_t bits_from(int begin, int first) { return from_bits(begin, first); }
int begin_of(const uint64_t* words, int count, int prefix, int nodes, int window) { return tree_begin(words, count, prefix, nodes, window); }
int begin_of_chain(int node, int prefix, int window) { return chain_begin(node, prefix, window); }
void draft(int32_t start, int32_t stop, int64_t rows, int32_t length, int64_t most, int window, int unit, int group, int columns, int* out) {
  const Draft d = draft_of(start, stop, rows, length, most, window, unit, group, columns);
  int* o = out;
  *o++ = d.row, *o++ = d.nodes, *o++ = d.prefix, *o++ = d.end, *o++ = d.unit, *o++ = d.units, *o++ = d.tiles;
}
uint32_t item_work() { return kItem; }
uint32_t work(int units, int tiles) {
  Draft d{};
  d.units = units, d.tiles = tiles;
  return work_of(d);
}
void share(uint32_t first, uint32_t units, uint32_t at, uint32_t stop, uint32_t* out) {
  const Share s = share_of(first, units, at, stop);
  out[0] = s.from, out[1] = s.to;
}
uint32_t place(uint32_t worker, int begins) { return place_of_part(worker, begins != 0); }
void parts(uint32_t first, uint32_t units, uint32_t per, uint32_t* out) {
  const TreeParts t = tree_parts(first, units, per);
  out[0] = t.from, out[1] = t.count;
}
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    path = tmp_path_factory.mktemp("tree")
    (path / "tree.cpp").write_text(SOURCE)
    subprocess.run([compiler, "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC",
                    f"-I{CSRC}", "-o", str(path / "tree.so"), str(path / "tree.cpp")], check=True)
    lib = ctypes.CDLL(str(path / "tree.so"))
    lib.bits_of.restype = lib.bits_of_chain.restype = lib.bits_from.restype = ctypes.c_uint32
    lib.draft.argtypes = [ctypes.c_int32, ctypes.c_int32, ctypes.c_int64, ctypes.c_int32, ctypes.c_int64] + [ctypes.c_int] * 4 + [ctypes.c_void_p]
    return lib


def test_bits(plan):
    """All 32 tokens from any node on, words that end inside them."""
    rng = np.random.default_rng(0)
    for words in (1, 2, 3):
        for _ in range(20):
            mask = rng.integers(-2 ** 63, 2 ** 63 - 1, words, dtype=np.int64)
            seen = np.concatenate([np.ones(80, bool), np.unpackbits(mask.astype("<i8").view(np.uint8), bitorder="little"), np.zeros(80, bool)])
            for first in range(-70, 64 * words + 70):
                want = int(sum(1 << x for x in range(32) if 0 <= 80 + first + x < len(seen) and seen[80 + first + x]))
                assert plan.bits_of(mask.ctypes.data_as(ctypes.c_void_p), words, first) == want, (words, first)
    for node in range(0, 70):
        for first in range(-70, 110):
            assert plan.bits_of_chain(node, first) == sum(1 << x for x in range(32) if first + x <= node)
    for begin in range(0, 80):
        for first in range(0, 100):
            assert plan.bits_from(begin, first) == sum(1 << x for x in range(32) if first + x >= begin)


@pytest.mark.parametrize("seed", range(8))
def test_windows(plan, seed):
    """The first token of the last `window` that a row sees, trees deeper than the window and caches shorter than the step among them."""
    rng = np.random.default_rng(seed)
    for _ in range(60):
        n, words = int(rng.integers(1, 150)), int(rng.integers(1, 4))
        length = int(rng.choice([rng.integers(1, n + 1), n + rng.integers(0, 100)]))
        mask = drafts.random_tree(rng, n, words, whole=bool(rng.integers(2)))
        mask |= np.where(rng.random(mask.shape) < 0.2, rng.integers(-2 ** 63, 2 ** 63 - 1, mask.shape), 0)  # (bits beyond the nodes too)
        for i in rng.integers(0, n, 6):
            row = np.ascontiguousarray(mask[i])
            for window in (1, 2, 5, int(rng.integers(1, 200)), 2 ** 31 - 1):
                seen = np.flatnonzero(drafts.sees(row, i, n, length, 0))[-window:]
                begin = plan.begin_of(row.ctypes.data_as(ctypes.c_void_p), words, length - n, n, window)
                got = np.flatnonzero(drafts.sees(row, i, n, length, 0))
                assert np.array_equal(got[got >= begin], seen), (n, words, length, i, window)
                chain = np.flatnonzero(drafts.sees(None, i, n, length, 0))
                begin = plan.begin_of_chain(int(i), length - n, window)
                assert np.array_equal(chain[chain >= begin], chain[-window:])


def test_drafts(plan):
    """A sequence's rows stay within the step's, its tokens within the table, and its units hold all that its rows may see."""
    rng = np.random.default_rng(1)
    out = np.zeros(7, np.int32)
    ends = [-2 ** 31, -1, 0, 1, 5, 64, 100, 2 ** 31 - 1]
    for _ in range(4000):
        start, stop, length = (int(rng.choice(ends)) for _ in range(3))
        rows, most = int(rng.choice([1, 5, 80])), int(rng.choice([0, 1, 64, 100, 1000]))
        window, unit, group, columns = int(rng.choice([0, 1, 7, 64, 2 ** 31 - 1])), int(rng.choice([64, 128])), int(rng.choice([1, 3, 16])), 16
        plan.draft(start, stop, rows, length, most, window, unit, group, columns, out.ctypes.data_as(ctypes.c_void_p))
        row, nodes, prefix, end, first, units, tiles = (int(x) for x in out)
        assert 0 <= row <= rows and 0 <= nodes and row + nodes <= rows
        assert end == min(max(length, 0), most) and prefix == end - nodes
        assert tiles == -(-nodes * group // columns)
        if nodes and end:
            assert (first + units) * unit >= end > (first + units - 1) * unit and first >= 0
            lowest = max(0, prefix - window) if window else 0  # a row that sees none of the step's own tokens
            assert first * unit <= lowest and (first + 1) * unit > lowest
        else:
            assert units == 0
    plan.draft(2, 7, 100, 50, 1000, 0, 128, 4, 16, out.ctypes.data_as(ctypes.c_void_p))
    assert out.tolist() == [2, 5, 45, 50, 0, 1, 2]


@pytest.mark.parametrize("seed", range(6))
def test_shares(plan, seed):
    """Every unit of every item goes to one worker; the workers of an item are those that its parts name, and no two parts lie in one
    place."""
    rng = np.random.default_rng(seed)
    out = np.zeros(2, np.uint32)
    at = out.ctypes.data_as(ctypes.c_void_p)
    plan.place.restype = plan.work.restype = plan.item_work.restype = ctypes.c_uint32
    way = plan.item_work()
    for _ in range(40):
        items = [int(x) for x in rng.integers(1, int(rng.choice([2, 6, 300])), int(rng.choice([1, 3, 40])))]
        assert plan.work(items[0], 3) == 3 * (items[0] + way) and plan.work(0, 3) == 0
        begins = np.concatenate([[0], np.cumsum([n + way for n in items])])
        workers = int(rng.choice([1, 2, 7, 64, 512]))
        per = -(-int(begins[-1]) // workers)
        places = set()
        for first, n in zip(begins.tolist(), items):
            plan.parts(first, n, per, at)
            start, count = (int(x) for x in out)
            have, covered = [], 0
            for w in range(workers):
                if (w + 1) * per <= first or w * per >= first + n + way:
                    continue
                plan.share(first, n, w * per, (w + 1) * per, at)
                lo, hi = (int(x) for x in out)
                if lo >= hi:
                    continue
                assert lo == covered and hi <= n
                covered = hi
                have.append(w)
                if hi - lo < n:
                    place = plan.place(w, lo == 0)
                    assert place not in places and place < 2 * workers
                    places.add(place)
            assert covered == n and have == list(range(start, start + count))
