"""The 8-bit product's kernels wait for counts of loads (vmcnt) that hold if each step issues the loads that its source
names and no fewer: this compiles transmuter_amd/csrc/tmh_fp8.hip to assembly and counts them."""

import os
import re
import shutil
import subprocess

import pytest

from transmuter_amd import build

SOURCE = os.path.join(build.CSRC, "tmh_fp8.hip")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Each kernel's template arguments and its sequence of waits: (name, arguments) -> [(loads to registers, to LDS, vmcnt or
    None, barrier)], the loads being those since the entry before."""
    if shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("no HIP compiler")
    out = tmp_path_factory.mktemp("fp8") / "fp8.s"
    subprocess.run([build.hipcc(), *build.COMMON, "--cuda-device-only", "-S", SOURCE, "-o", str(out)], check=True, capture_output=True)
    found, key = {}, None
    for line in out.read_text().splitlines():
        start = re.match(r"_ZN\S*?(k_f8_gemm|k_f8_rows)I((?:L[ib]\d+E)+)E\S*:", line)
        if start:
            key = (start[1], tuple(int(v) for v in re.findall(r"L[ib](\d+)E", start[2])))
            found[key], loads = [], [0, 0]
        if key is None:
            continue
        text = line.strip()
        if re.match(r"(buffer|global)_load", text):
            loads[" lds" in text] += 1
        wait = re.match(r"s_waitcnt .*vmcnt\((\d+)\)", text)
        if wait or text.startswith("s_barrier"):
            found[key].append((*loads, int(wait[1]) if wait else None, text.startswith("s_barrier")))
            loads = [0, 0]
        if text.startswith("s_endpgm"):
            key = None
    assert found
    return found


def test_tiles(kernels):
    seen = 0
    for (name, args), waits in kernels.items():
        if name != "k_f8_gemm":
            continue
        bm, bn, wm, wn, dw, da, _exact, touch = args
        weights, rows = 2 * (bn // 16 // wn) + 1, 2 * (bm // 16) // (wm * wn) + 1
        # In front of the first step, and with each step behind its wait and barrier.
        first, step = (dw * weights, da * rows + dw * touch), (weights, rows + touch)
        count = (dw - 1) * (weights + rows + touch) + (rows if da > dw else 0) + touch
        steps = [i for i, w in enumerate(waits[:-1]) if w[2] == count and waits[i + 1] == (0, 0, None, True)]
        assert len(steps) == dw + 1, (args, waits)
        assert waits[steps[0]][:2] == first, (args, waits)
        assert all(waits[i][:2] == step for i in steps[1:]), (args, waits)
        # The last step's loads; then everything is waited for ahead of the steps without loads.
        rest = waits[steps[-1] + 2:]
        assert rest[0][:2] == step and (0, 0, None, True) in rest
        assert rest[rest.index((0, 0, None, True)) - 1][2] == 0 and all(w[:2] == (0, 0) for w in rest[1:rest.index((0, 0, None, True))])
        seen += 1
    assert seen >= 4


def test_rows(kernels):
    seen = 0
    for (name, args), waits in kernels.items():
        if name != "k_f8_rows":
            continue
        mt, nt, _kw, depth, _exact = args
        registers, lds = 2 * nt + 1 + mt, 2 * mt
        for ahead in range(1, depth):
            here = [w for w in waits if w[2] == ahead * (registers + lds)]
            assert here, (args, waits)
            if ahead == depth - 1:  # behind a block's own loads; fewer are waited for where there are no more
                assert all(w[:2] == (registers, lds) for w in here), (args, waits)
        seen += 1
    assert seen >= 4
