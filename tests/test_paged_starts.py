"""Rows matched to sequences whose starts may be anything, on the CPU (csrc/mmnb_paged_plan.h
built for the host)."""
import ctypes
import functools
import itertools
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
// place of row t in sequence b (-1: not one of its rows), and whether the sequence is bad
int place(const int32_t *start, const int32_t *len, int b, int t, int tokens, int *bad) {
  const PagedSeq s = paged_seq(start[b], start[b + 1], len[b], tokens, tokens, 100);
  *bad = s.bad;
  return paged_in(s, t) ? t - s.row0 : -1;
}
int holds(const int32_t *start, int b, int t) { return paged_holds(start, b, t); }
}
"""


@functools.lru_cache(None)
def lib():
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = Path(tempfile.mkdtemp())
    (d / "starts.cpp").write_text(SHIM)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-O1", "-shared", "-fPIC", "-I",
                    str(CSRC), str(d / "starts.cpp"), "-o", str(d / "starts.so")], check=True)
    return ctypes.CDLL(str(d / "starts.so"))


TOKENS = 6


@pytest.mark.parametrize("lens", [(100, 100, 100), (4, 2, 0), (0, 3, 100)])
def test_a_sequence_found_by_any_search_only_takes_rows_of_its_own(lens):
    """Keys of a row lie in its sequence, whatever sequence a search of the starts has found."""
    n = ctypes.c_int32 * 3
    bad = ctypes.c_int()
    for start in itertools.product((-2, 0, 1, 3, 4, 6, 9), repeat=4):
        s, ln = (ctypes.c_int32 * 4)(*start), n(*lens)
        for t in range(TOKENS):
            for b in range(3):
                i = lib().place(s, ln, b, t, TOKENS, ctypes.byref(bad))
                own = start[b] <= t < start[b + 1]
                assert bool(lib().holds(s, b, t)) == own == (i >= 0)
                if own and not bad.value:
                    rows = start[b + 1] - start[b]
                    assert i == t - start[b] and 0 <= lens[b] - rows + i < lens[b]


def test_a_row_before_its_sequence_has_no_place_in_it():
    """Row 1 of starts 3, 4, 1 lies behind one start, as a row of the first sequence would."""
    bad = ctypes.c_int()
    s, ln = (ctypes.c_int32 * 3)(3, 4, 1), (ctypes.c_int32 * 2)(10, 5)
    for t in (1, 2):
        assert sum(x <= t for x in s) == 1
        assert lib().place(s, ln, 0, t, 4, ctypes.byref(bad)) == -1 and not bad.value
    assert lib().place(s, ln, 0, 3, 4, ctypes.byref(bad)) == 0
