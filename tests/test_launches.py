"""How work is cut into launches (transmuter_amd/csrc/tmh_launch.h) on the host: every thing once, no grid with more threads
than HIP takes."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transmuter_amd", "csrc")

# (test code only: what it compiles is the header that the launches include)
SOURCE = r"""
#include "tmh_launch.h"
extern "C" int64_t runs(int64_t all, int threads, int64_t per, int64_t pieces, int64_t most, int64_t* out) {
  int64_t n = 0;
  tmh::in_launches(all, tmh::most_a_launch(threads, per, pieces), [&](int64_t first, int64_t count) {
    if (n < most) out[2 * n] = first, out[2 * n + 1] = count;
    ++n;
  });
  return n;
}
"""


@pytest.fixture(scope="module")
def runs(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    path = tmp_path_factory.mktemp("launch")
    (path / "launch.cpp").write_text(SOURCE)
    subprocess.run([compiler, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", "-o",
                    str(path / "launch.so"), str(path / "launch.cpp")], check=True)
    lib = ctypes.CDLL(str(path / "launch.so"))
    lib.runs.argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p]
    lib.runs.restype = ctypes.c_int64

    def call(all, threads, per, pieces):
        out = np.zeros((4096, 2), np.int64)
        n = lib.runs(all, threads, per, pieces, len(out), out.ctypes.data)
        assert n <= len(out)
        return [(int(a), int(b)) for a, b in out[:n]]

    return call


# Threads, pieces a workgroup takes, pieces of one thing: rows of the norm (four to a workgroup, one to one of 64 to 1024
# threads), blocks of 128 of rows in 8 bits, 16-byte pieces of padded rows, tiles of a weight.
SHAPES = [(256, 4, 1), (64, 1, 1), (128, 1, 1), (1024, 1, 1), (256, 16, 1), (256, 16, 86), (256, 16, 2 ** 23), (256, 256, 1), (256, 4, 1)]


@pytest.mark.parametrize("threads,per,pieces", SHAPES)
@pytest.mark.parametrize("all", [0, 1, 3, 4, 5, 2 ** 20 + 1, 2 ** 22 - 1, 2 ** 22, 2 ** 26, 2 ** 26 + 1, 2 ** 28, 2 ** 28 + 5, 2 ** 31 - 1])
def test_launches(runs, all, threads, per, pieces):
    if all // max(1, 2 ** 24 * per // pieces) > 4000:
        all %= 2 ** 16
    got = runs(all, threads, per, pieces)
    at = 0
    for i, (first, count) in enumerate(got):
        assert first == at and count > 0
        groups = -(-count * pieces // per)
        assert groups * threads < 2 ** 32
        assert count * pieces < 2 ** 31 or per == 256  # the quantizer's divisions
        assert pieces > 1 or count % per == 0 or i == len(got) - 1  # no workgroup of one launch reaches into the next
        at += count
    assert at == all
    # One launch where one does.
    if -(-all * pieces // per) * threads < 2 ** 32 - threads * pieces:
        assert len(got) <= 1
