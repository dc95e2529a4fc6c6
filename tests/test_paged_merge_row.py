"""The layout of the merge's rows in LDS, on the CPU."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "onnx_runtime_dart_amd" / "csrc"
SHIM = """
#include "mmnb_paged_plan.h"
#include <cstdio>
int main() { std::printf("%d %d", mmnb::kPagedMergeRow, (int)mmnb::kPagedMaxHead); }
"""


def test_every_wave_stores_vectors_of_four_at_their_alignment(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    (tmp_path / "row.cpp").write_text(SHIM)
    subprocess.run([cxx, "-std=c++17", "-I", str(CSRC), str(tmp_path / "row.cpp"), "-o",
                    str(tmp_path / "row")], check=True)
    row, head = map(int, subprocess.run([str(tmp_path / "row")], check=True,
                                        capture_output=True).stdout.split())
    assert row >= head + 2                       # the sums, m and l
    for wave in range(4):
        for d in range(0, head, 4):              # stored 16 bytes at a time
            assert (wave * row + d) * 4 % 16 == 0
    # and in the kernel
    src = (CSRC / "mmnb_paged_attn.h").read_text()
    assert "__attribute__((aligned(16))) float sm[4][kPagedMergeRow]" in src
