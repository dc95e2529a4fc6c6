"""Where append may write the turned queries, on the CPU."""
import ctypes
import functools
import itertools
import shutil
import subprocess
import tempfile
import types
from pathlib import Path

import pytest

from onnx_runtime_dart_amd import _lib, paged

CSRC = Path(__file__).resolve().parents[1] / "onnx_runtime_dart_amd" / "csrc"
SHIM = """
#include "mmnb_paged_plan.h"
using namespace mmnb;
extern "C" int in_place(int64_t in, int64_t ldi, int64_t out, int64_t ldo, int64_t w, int64_t n) {
  return paged_check_in_place((const float *)in, ldi, (const float *)out, ldo, w, n).code;
}
"""


@functools.lru_cache(None)
def lib():
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = Path(tempfile.mkdtemp())
    (d / "place.cpp").write_text(SHIM)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-O1", "-shared", "-fPIC", "-I",
                    str(CSRC), str(d / "place.cpp"), "-o", str(d / "place.so")], check=True)
    f = ctypes.CDLL(str(d / "place.so")).in_place
    f.argtypes = [ctypes.c_int64] * 6
    return f


def test_rows_take_their_own_place_or_none():
    """Refused where a row's place is another's in part; and never refused where all rows are
    apart, but for strides that differ (whose rows might lie between each other's)."""
    w = 4
    for rows, ldi, ldo, off in itertools.product((1, 2, 3), (4, 6, 9), (4, 6, 9), range(-40, 41)):
        a = [set(range(t * ldi, t * ldi + w)) for t in range(rows)]
        b = [set(range(off + t * ldo, off + t * ldo + w)) for t in range(rows)]
        safe = all(not (x & y) or (i == j and x == y)
                   for i, x in enumerate(a) for j, y in enumerate(b))
        code = lib()(4096, ldi, 4096 + 4 * off, ldo, w, rows)
        if not safe:
            assert code == _lib.MMNB_ERR_ARG, (rows, ldi, ldo, off)
        elif ldi == ldo or off >= rows * ldi or -off >= rows * ldo:
            assert code == 0, (rows, ldi, ldo, off)


@pytest.mark.parametrize("kw,want", [
    (dict(q=4096, q_out=4096, ldq=1000), 1000), (dict(q=4096, q_out=4096), 128),
    (dict(q=4096, q_out=8192, ldq=1000), 128), (dict(q=4096, q_out=4096, ldq=1000, ldqo=500), 500),
    (dict(q=None, q_out=None, ldq=1000), 1000)])
def test_queries_turned_in_place_keep_their_row_stride(kw, want):
    seen = []
    so = types.SimpleNamespace(mmnb_paged_append_dev=lambda *a: seen.append(a) or 0)
    ctx = types.SimpleNamespace(lib=so, handle=None)
    cache = paged.PagedCache(4096, 8192, "f16", num_pages=1, page_size=16, kv_heads=1,
                             head_size=64)
    batch = paged.PagedBatch(0, 0, 0, batch=1, tokens=1, page_cols=1, max_q=1, max_kv=16)
    q, q_out = kw.pop("q"), kw.pop("q_out")
    paged.append(cache, batch, q, 4096, 4096, 4096, 4096, q_out, heads=2, max_pos=16, half_rot=32,
                 ctx=ctx, **kw)
    assert seen[0][-1] == want


def test_strides_and_rows_as_large_as_they_may_be():
    big = 1 << 40
    assert lib()(4096, big, 4096, big, 4, 1 << 30) == 0
    assert lib()(4096, big, 4096, big - 1, 4, 1 << 30) == _lib.MMNB_ERR_ARG
    assert lib()(4096, big, 1 << 62, 4, 4, 1 << 30) == _lib.MMNB_ERR_ARG
    assert lib()(1 << 62, 4, 4096, 4, 4, 1 << 30) == 0
