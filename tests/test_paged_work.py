"""How paged attention's work is dealt out, on the CPU (csrc/mmnb_paged_plan.h built for the
host)."""
import ctypes
import functools
import shutil
import subprocess
import tempfile
from pathlib import Path

import pytest

from onnx_runtime_dart_amd import _lib

CSRC = Path(__file__).resolve().parents[1] / "onnx_runtime_dart_amd" / "csrc"
SHIM = """
#include "mmnb_paged_plan.h"
using namespace mmnb;
extern "C" {
int64_t each(int64_t t, int64_t most) { return paged_each((int)t, (int)most); }
int size(const mmnb_paged_batch *b, int64_t heads) { return paged_check_size(*b, heads).code; }
void range(int n, int len, int bad, int window, int two, int tile, int *o) {
  const PagedRange r = paged_range({0, n, len, bad != 0}, window, two, tile);
  o[0] = r.lo, o[1] = r.n;
}
void keys(int n, int len, int prefix, int group, int window, int two, int first, int count,
          int tile, int *o) {
  const PagedKeys k = paged_keys({0, n, len, false}, prefix, group, window, two, first, count,
                                 tile);
  o[0] = k.loa, o[1] = k.na, o[2] = k.lob, o[3] = k.nb, o[4] = k.own;
}
int tiles_of(int n, int bad, int group, int rows) {
  return paged_tiles_of({0, n, n, bad != 0}, group, rows);
}
int64_t parts(int64_t b, int64_t t, int64_t g, int64_t bytes, int64_t most) {
  return paged_prompt_parts(b, t, g, bytes, most);
}
int seen(int p, int w, int two) { return paged_prefix_seen(p, w, two != 0); }
int behind(int n, int len, int bad, int group, int rows, int x) {
  return paged_tiles_behind({0, n, len, bad != 0}, group, rows, x);
}
int64_t row_tiles(int64_t b, int64_t t, int64_t q, int64_t g, int64_t r) {
  return paged_row_tiles(b, t, q, g, r);
}
int64_t splits(int64_t b, int64_t t, int64_t l, int64_t c) { return paged_splits(b, t, l, c); }
}
"""


@functools.lru_cache(None)
def lib():
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tempfile.mkdtemp()
    src, so = Path(d) / "work.cpp", Path(d) / "work.so"
    src.write_text(SHIM)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-O1", "-shared", "-fPIC", "-I",
                    str(CSRC), str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    for name, n in (("each", 2), ("row_tiles", 5), ("splits", 4), ("parts", 5)):
        f = getattr(lib, name)
        f.restype, f.argtypes = ctypes.c_int64, [ctypes.c_int64] * n
    return lib


@pytest.mark.parametrize("total", [1, 2, 7, 136, 1023, 1024, 1025, 5000, (1 << 31) - 1])
@pytest.mark.parametrize("most", [1, 3, 512, 1024])
def test_the_waves_take_all_tiles(total, most):
    each = lib().each(total, most)
    assert each * most >= total > (each - 1) * most


def test_rows_past_32_bits_are_refused():
    b = _lib.PagedBatch(1, 1 << 30, None, None, None, 1 << 30, 1 << 30, 1 << 30)
    assert lib().size(ctypes.byref(b), ctypes.c_int64(1)) == 0
    assert lib().size(ctypes.byref(b), ctypes.c_int64(2)) == _lib.MMNB_ERR_UNSUPPORTED
    b.tokens = (1 << 24) - 1
    assert lib().size(ctypes.byref(b), ctypes.c_int64(127)) == 0
    assert lib().size(ctypes.byref(b), ctypes.c_int64(128)) == _lib.MMNB_ERR_UNSUPPORTED


@pytest.mark.parametrize("window", [0, 1, 5, 40, 1000])
@pytest.mark.parametrize("n,length", [(1, 1), (1, 33), (3, 100), (40, 64), (8, 8)])
@pytest.mark.parametrize("two", [-5, 0, 7])
@pytest.mark.parametrize("tile", [32, 64])
def test_the_range_holds_every_key_that_a_row_sees(window, n, length, two, tile):
    o = (ctypes.c_int * 2)()
    lib().range(n, length, 0, window, two, tile, o)
    lo, tiles = o
    seen = {j for i in range(length - n, length) for j in range(length)
            if (j <= i and (not window or i - j < window)) or j < two}
    assert lo % tile == 0 and lo >= 0 and tiles >= 1
    assert min(seen) >= lo and max(seen) < lo + tiles * tile < length + tile
    if window and two <= 0:
        assert min(seen) < lo + tile


def test_sequences_without_rows_have_no_tiles_and_broken_ones_one():
    o = (ctypes.c_int * 2)()
    lib().range(0, 50, 0, 0, 0, 32, o)
    assert o[1] == 0
    lib().range(5, 0, 1, 0, 0, 32, o)
    assert o[1] == 1


@pytest.mark.parametrize("new", [[1], [700, 3, 1, 0, 64], [128] * 9, [33, 31], [5] * 50])
@pytest.mark.parametrize("group", [1, 2, 3, 8])
@pytest.mark.parametrize("rows", [64, 128])
def test_row_tiles_suffice(new, group, rows):
    need = sum(-(-n * group // rows) for n in new)
    got = lib().row_tiles(len(new), sum(new), max(new), group, rows)
    assert need <= got <= need + len(new) * max(1, -(-max(new) * group // rows))


def test_splits():
    assert lib().splits(2048, 128, 1, 512) == 1
    assert lib().splits(8, 128, 1, 512) == 64
    assert lib().splits(8, 3, 1, 512) == 3
    assert lib().splits(12, 63, 1, 512) == 32  # two tiles each, where 42 parts leave some empty
    assert lib().splits(100, 1000, 1, 512) == 5
    assert lib().splits(424, 1000, 1, 512) == 1
    assert lib().splits(32, 63, 8, 512) == 7
    assert lib().splits(24, 354, 16, 256) == 10
    assert lib().splits(128, 5, 8, 512) == 1
    assert lib().splits(1, 1, 1, 512) == 1


ROWS = [(n, length, group, first, count)
        for n, length in ((1, 1), (3, 100), (70, 200), (200, 200))
        for group, first, count in ((1, 0, 128), (4, 0, 128), (3, 128, 128), (1, 64, 32))
        if first < n * group]


@pytest.mark.parametrize("prefix", [0, 5, 64, 100])
@pytest.mark.parametrize("n,length,group,first,count", ROWS)
@pytest.mark.parametrize("window", [0, 1, 9, 90])
@pytest.mark.parametrize("two", [0, 3, 80, 250])
def test_the_tiles_hold_the_keys_that_the_rows_see(prefix, n, length, group, first, count, window,
                                                   two):
    o = (ctypes.c_int * 5)()
    lib().keys(n, length, prefix, group, window, two, first, count, 64, o)
    loa, na, lob, nb, own = o
    seen = set()
    for i in {k // group for k in range(first, min(first + count, n * group))}:
        p = prefix + length - n + i
        seen |= {j for j in range(prefix + length)
                 if (j <= p and (not window or p - j < window)) or j < two}
    a = {j for j in seen if j < prefix}
    b = {j - prefix for j in seen if j >= prefix}
    assert loa % 64 == 0 and lob % 64 == 0 and na >= 0 and nb >= 0
    assert a <= set(range(loa, min(prefix, loa + 64 * na)))
    assert b <= set(range(lob, min(own, lob + 64 * nb))) and own == max(b, default=-1) + 1
    assert na + nb >= 1 and (not na or loa + 64 * (na - 1) < prefix)
    assert not nb or lob + 64 * (nb - 1) < own <= length


def test_tiles_of_a_sequence():
    assert [lib().tiles_of(n, 0, 3, 128) for n in (0, 1, 42, 43, 128)] == [0, 1, 1, 2, 3]
    assert lib().tiles_of(500, 1, 3, 128) == 1 and lib().tiles_of(0, 1, 3, 128) == 0


@pytest.mark.parametrize("group", [1, 3, 8, 200])
@pytest.mark.parametrize("rows", [64, 128])
@pytest.mark.parametrize("n,length", [(1, 1), (5, 40), (130, 130), (300, 1000)])
def test_tiles_that_end_behind_a_key(n, length, group, rows):
    tiles = -(-n * group // rows)
    ends = [length - n + min(n, ((t + 1) * rows - 1) // group + 1) for t in range(tiles)]
    assert ends[-1] == length
    for x in range(-1, length + 2):
        assert lib().behind(n, length, 0, group, rows, x) == sum(e > x for e in ends)


def test_broken_sequences_come_last():
    assert [lib().behind(7, 0, 1, 2, 64, x) for x in (-1, 0, 1, 5)] == [1, 1, 0, 0]
    assert lib().behind(0, 0, 1, 2, 64, -1) == 0


@pytest.mark.parametrize("prefix", [1, 64, 65, 1000])
@pytest.mark.parametrize("window", [0, 1, 2, 64, 130, 999, 1000, 5000])
def test_prefix_keys_that_no_row_sees(prefix, window):
    lo = lib().seen(prefix, window, 0)
    assert lo % 64 == 0 and 0 <= lo < prefix and lib().seen(prefix, window, 1) == 0
    # the first row behind the prefix sees the most of it
    sees = [j for j in range(prefix) if not window or prefix - j < window]
    assert not sees or min(sees) >= lo
    assert not window or window >= prefix or prefix - window + 1 - lo < 128


def test_parts_of_a_prompts_keys():
    row = 130 * 4
    assert lib().parts(32, 63, 2, 64 * 32 * row, 256) == 8      # all that fit
    assert lib().parts(128, 16, 2, 256 * 32 * row, 256) == 1    # not worth a merge
    assert lib().parts(128, 63, 2, 256 * 32 * row, 256) == 2
    assert lib().parts(257, 5000, 1, 0, 512) == 1
    assert 4 <= lib().parts(6, 34, 2, 27 * 8 * row, 256) <= 17
    assert lib().parts(1, 1, 2, 0, 256) == 1
    for tiles in (2, 3, 7, 100):
        assert 1 <= lib().parts(1, tiles, 2, 0, 256) <= tiles // 2 + 1
