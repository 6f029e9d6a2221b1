"""The 8-bit product's choice of kernel and parts of K (transmuter_amd/csrc/tmh_fp8_plan.h) on the host: grids within what HIP
takes, every kernel reached, and the GPU tests' sizes in each of them, whole and in parts, in both kinds of answer."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import test_gpu_fp8_shapes as shapes
import test_gpu_serving as base
import test_gpu_serving_norms as norms

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transmuter_amd", "csrc")
CUS = 256
KERNELS = ["ROWS16", "ROWS16_WIDE", "ROWS32_WIDE", "ROWS64", "GEMM_64x64", "GEMM_64x128", "GEMM_128x128", "GEMM_128x256"]

# (test code only: what it compiles is the header that the product includes)
SOURCE = r"""
#include "tmh_fp8_plan.h"
using namespace tmh;
static_assert(ROWS16 == 0 && ROWS64 == 3 && GEMM_128x256 == 7, "the order of the names");
extern "C" void plan(int64_t M, int64_t N, int64_t K, int f32, int cus, int* out) {
  const int kb = static_cast<int>((K + 127) / 128);
  const F8Plan p = plan_of(M, N, kb, (N + 31) / 32 * 2, f32 != 0, cus);
  out[0] = p.kernel;
  out[1] = p.splits;
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
    f.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] * 2 + [ctypes.c_void_p]

    def call(m, k, n, f32):
        out = (ctypes.c_int * 2)()
        f(m, n, k, int(f32), CUS, out)
        blocks = -(-k // 128)
        per = -(-blocks // out[1])
        return KERNELS[out[0]], -(-blocks // per)

    return call


def grid_threads(kernel, m, n):
    if kernel.startswith("ROWS"):
        rows, cols = {"ROWS16": (16, 16), "ROWS16_WIDE": (16, 32), "ROWS32_WIDE": (32, 32), "ROWS64": (64, 16)}[kernel]
        return -(-n // 32) * 32 // cols * -(-m // rows) * 512
    bm, bn = (int(v) for v in kernel[5:].split("x"))
    return -(-n // bn) * -(-m // bm) * 256


@pytest.mark.parametrize("f32", [False, True])
def test_plans(plan, f32):
    rng = np.random.default_rng(int(f32))
    seen = set()
    for m, k, n in zip(*(np.maximum(1, 2 ** rng.uniform(0, top, 60000)).astype(np.int64).tolist() for top in (22, 17, 22))):
        if m * n > 2 ** 37 or m * k > 2 ** 38 or k * n > 2 ** 38:
            continue  # (more than the card's memory)
        kernel, parts = plan(m, k, n, f32)
        assert 1 <= parts <= 8 and (parts == 1 or kernel.startswith("GEMM")) and not (f32 and kernel == "GEMM_128x256")
        assert grid_threads(kernel, m, n) < 2 ** 32, (m, k, n, kernel)
        seen.add((kernel, parts > 1))
    tiles = KERNELS[4:7] if f32 else KERNELS[4:]
    assert seen == {(v, False) for v in KERNELS[:4]} | {(v, parts) for v in tiles for parts in (False, True)}


def test_gpu_sizes(plan):
    """The GPU tests' sizes reach each kernel, whole and in parts of K; of the sizes compared in the 2-norm each kernel has some
    of twelve blocks of K or more, and the widest tile both with few bytes and with those that its look-ahead is for."""
    every = {(f32, v, False) for f32 in (False, True) for v in KERNELS[:4]}
    every |= {(f32, v, parts) for f32 in (False, True) for v in KERNELS[4:] for parts in (False, True) if not (f32 and v == "GEMM_128x256")}
    seen, deep, touched = set(), set(), set()
    for m, k, n in norms.PRODUCTS:
        for f32 in (False, True):
            kernel, parts = plan(m, k, n, f32)
            seen.add((f32, kernel, parts > 1))
            if -(-k // 128) >= 12:
                deep.add(kernel)
                if kernel == "GEMM_128x256" and parts == 1:
                    touched.add(m * k + n * k + 2 * m * n > 90e6)
    assert seen == every, every - seen
    assert deep >= set(KERNELS) - {"ROWS64"}
    for m, k, n in shapes.SHAPES + base.PRODUCTS:
        for f32 in (False, True):
            kernel, parts = plan(m, k, n, f32)
            seen.add((f32, kernel, parts > 1))
    assert seen == every and touched == {False, True}
