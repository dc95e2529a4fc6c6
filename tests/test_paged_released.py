"""Page numbers that rows need, and those before their windows, on the CPU
(csrc/mmnb_paged_plan.h built for the host)."""
import ctypes
import functools
import shutil
import subprocess
import tempfile
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "onnx_runtime_dart_amd" / "csrc"
SHIM = """
#include "mmnb_paged_plan.h"
using namespace mmnb;
extern "C" {
void span(int p, int window, int two, int keys, int *o) {
  const PagedSpan s = paged_row_span(p, window, two, keys);
  o[0] = s.lo, o[1] = s.hi;
}
// pages lost one after the other (and others that are not), and whether they are missed
int missed(int n, const int *pages, int shift, int off, int p, int window, int two) {
  int l = -1;
  for (int i = 0; i < n; i++) {
    l = paged_lose(l, true, pages[i], shift, off);
    l = paged_lose(l, false, 5, shift, off);
  }
  return paged_missed(l, shift, p, window, two);
}
}
"""


@functools.lru_cache(None)
def lib():
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = Path(tempfile.mkdtemp())
    (d / "r.cpp").write_text(SHIM)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-O1", "-shared", "-fPIC", "-I",
                    str(CSRC), str(d / "r.cpp"), "-o", str(d / "r.so")], check=True)
    return ctypes.CDLL(str(d / "r.so"))


def sees(p, window, two, total):
    return [j for j in range(total) if (j <= p and (not window or p - j < window)) or j < two]


def test_keys_of_a_row():
    o = (ctypes.c_int * 2)()
    for p in (0, 1, 20, 99):
        for window in (0, 1, 7, 50, 500):
            for two in (0, 3, 60, 500):
                lib().span(p, window, two, 100, o)
                seen = sees(p, window, two, 100)
                assert o[0] <= min(seen) and o[1] == max(seen) + 1
                assert two or o[0] == min(seen)


@pytest.mark.parametrize("shift,off", [(0, 0), (2, 0), (3, 7), (4, 100)])
def test_rows_miss_what_they_see_of_the_pages_that_are_lost(shift, off):
    size, total = 1 << shift, off + (6 << shift)
    for lost in ([], [0], [1], [0, 3], [5], [4, 1], [2, 3]):
        keys = {off + k for page in lost for k in range(page * size, (page + 1) * size)}
        flat = (ctypes.c_int * (len(lost) + 1))(*lost)
        for p in (off, off + 5, total - 1):
            for window in (0, 1, 4, 17, 500):
                for two in (0, off + 1, off + 30):
                    got = lib().missed(len(lost), flat, shift, off, p, window, two)
                    first = p - window + 1 if window and p >= window else 0
                    want = bool(keys) and (two > 0 or max(keys) >= first)
                    assert bool(got) == want
                    # never less than what some row from p on sees
                    assert got or not keys & set(sees(p, window, two, total))
