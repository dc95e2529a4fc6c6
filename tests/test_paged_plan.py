"""What calls on a paged cache refuse, and how lengths and page numbers from the device are
made safe, on the CPU (csrc/mmnb_paged_plan.h built for the host)."""
import ctypes
import functools
import itertools
import shutil
import subprocess
import tempfile
from pathlib import Path

import pytest

from onnx_runtime_dart_amd import _lib, paged

CSRC = Path(__file__).resolve().parents[1] / "onnx_runtime_dart_amd" / "csrc"
SHIM = """
#include "mmnb_paged_plan.h"
using namespace mmnb;
extern "C" {
int cache(const mmnb_paged_cache *c) { return paged_check_cache(c).code; }
int batch(const mmnb_paged_cache *c, const mmnb_paged_batch *b) {
  return paged_check_batch(*c, b).code;
}
int rows(const mmnb_paged_cache *c, int64_t h, int64_t ld) {
  return paged_check_rows(*c, h, ld).code;
}
int rope(const mmnb_paged_cache *c, const mmnb_paged_batch *b, int tables, int64_t max_pos,
         int64_t half, int64_t first) {
  const float x = 0;
  return paged_check_rope(*c, *b, tables ? &x : nullptr, tables ? &x : nullptr, max_pos, half,
                          first).code;
}
int heads(const mmnb_paged_cache *c, int64_t h) { return paged_check_heads(*c, h).code; }
int scores(const mmnb_paged_scores *s) { return paged_check_scores(s).code; }
int prefix(const mmnb_paged_batch *b, int have, int64_t len) {
  const int32_t x = 0;
  return paged_check_prefix(*b, have ? &x : nullptr, len).code;
}
void strides(const mmnb_paged_cache *c, int64_t *o) {
  const PagedStrides s = paged_strides(*c);
  o[0] = s.page, o[1] = s.head, o[2] = s.row;
}
void seq(int s, int e, int len, int64_t tokens, int64_t mq, int64_t mk, int *o) {
  const PagedSeq q = paged_seq(s, e, len, tokens, mq, mk);
  o[0] = q.row0, o[1] = q.n, o[2] = q.len, o[3] = q.bad;
}
int page(int p, int n, int *bad) {
  bool b = *bad;
  const int r = paged_page(p, n, &b);
  *bad = b;
  return r;
}
}
"""
ARG, UNS = _lib.MMNB_ERR_ARG, _lib.MMNB_ERR_UNSUPPORTED


@functools.lru_cache(None)
def lib():
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not available")
    d = Path(tempfile.mkdtemp(prefix="paged_plan"))
    (d / "plan.cpp").write_text(SHIM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-I", str(CSRC),
                    str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    return ctypes.CDLL(str(d / "plan.so"))


I64 = ctypes.c_int64


def cache(**kw):
    c = _lib.PagedCache(0x1000, 0x2000, _lib.DT_F16, 10, 16, 2, 64, 0, 0, 0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def batch(**kw):
    b = _lib.PagedBatch(3, 7, 0x1000, 0x1000, 0x1000, 4, 5, 64)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(type=_lib.DT_F32), 0), (dict(type=_lib.DT_BF16), 0), (dict(type=2), UNS),
    (dict(num_pages=0), ARG), (dict(num_pages=1 << 31), UNS), (dict(page_size=0), ARG),
    (dict(page_size=48), UNS), (dict(page_size=1 << 17), UNS), (dict(page_size=1), 0),
    (dict(kv_heads=-1), ARG), (dict(kv_heads=1 << 16), UNS), (dict(head_size=0), ARG),
    (dict(head_size=60), UNS), (dict(head_size=136), UNS), (dict(head_size=8), 0),
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(v=0x2008), ARG), (dict(k=0x1002), ARG),
    (dict(stride_page=4096), ARG), (dict(stride_page=2048, stride_head=1024, stride_row=64), 0),
    (dict(stride_page=2048, stride_head=1024, stride_row=56), ARG),
    (dict(stride_page=2048, stride_head=1024, stride_row=68), UNS),
    (dict(stride_page=2044, stride_head=1024, stride_row=64), UNS),
    (dict(stride_page=-2048, stride_head=1024, stride_row=64), ARG),
    (dict(stride_page=1 << 41, stride_head=1024, stride_row=64), UNS)])
def test_caches(kw, code):
    assert lib().cache(ctypes.byref(cache(**kw))) == code


def test_null_structures():
    assert lib().cache(None) == ARG
    assert lib().batch(ctypes.byref(cache()), None) == ARG
    assert lib().scores(None) == 0


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(batch=-1), ARG), (dict(tokens=-1), ARG), (dict(page_cols=-1), ARG),
    (dict(max_q=-1), ARG), (dict(max_kv=-1), ARG), (dict(batch=70000), UNS),
    (dict(tokens=(1 << 30) + 1), UNS), (dict(max_kv=(1 << 30) + 1, page_cols=1 << 30), UNS),
    (dict(page_cols=1 << 31), UNS), (dict(max_q=65), ARG), (dict(max_kv=65), ARG),
    (dict(start=None), ARG), (dict(kv_len=None), ARG), (dict(pages=None), ARG),
    (dict(pages=None, max_kv=0, max_q=0), 0), (dict(batch=0, start=None, kv_len=None), 0),
    (dict(tokens=0, start=None), 0)])
def test_batches(kw, code):
    assert lib().batch(ctypes.byref(cache()), ctypes.byref(batch(**kw))) == code


@pytest.mark.parametrize("h,ld,code", [(4, 256, 0), (4, 255, ARG), (4, 300, 0), (0, 256, ARG),
                                       (70000, 1 << 30, ARG), (4, -256, ARG),
                                       (4, (1 << 40) + 1, UNS)])
def test_rows(h, ld, code):
    assert lib().rows(ctypes.byref(cache()), I64(h), I64(ld)) == code


@pytest.mark.parametrize("tables,max_pos,half,first,code", [
    (1, 64, 32, 0, 0), (1, 64, 33, 0, ARG), (1, 0, 32, 0, ARG), (0, 64, 32, 0, ARG),
    (0, 0, 0, 0, 0), (1, 64, -1, 0, ARG), (1, 64, 32, -1, ARG), (1, 64, 32, 1 << 30, UNS),
    (1, 1 << 40, 5, 1000, 0)])
def test_rotary(tables, max_pos, half, first, code):
    assert lib().rope(ctypes.byref(cache()), ctypes.byref(batch()), tables, I64(max_pos),
                      I64(half), I64(first)) == code


def test_heads():
    assert lib().heads(ctypes.byref(cache()), I64(6)) == 0
    assert lib().heads(ctypes.byref(cache()), I64(5)) == ARG


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG),
    (dict(softcap=-1.0), ARG), (dict(softcap=float("inf")), ARG), (dict(window=-1), ARG),
    (dict(window=1 << 60), 0), (dict(scale=-2.0), 0)])
def test_scores(kw, code):
    s = _lib.PagedScores(0.0, 0.0, 0, None, None)
    for k, v in kw.items():
        setattr(s, k, v)
    assert lib().scores(ctypes.byref(s)) == code


@pytest.mark.parametrize("have,n,code", [(1, 100, 0), (0, 0, 0), (0, 1, ARG), (1, -1, ARG),
                                         (1, 1 << 30, UNS), (1, (1 << 62), UNS)])
def test_prefixes(have, n, code):
    assert lib().prefix(ctypes.byref(batch()), have, I64(n)) == code


def test_default_strides():
    o = (I64 * 3)()
    lib().strides(ctypes.byref(cache()), o)
    assert list(o) == [2 * 16 * 64, 16 * 64, 64]


EDGES = [-(1 << 31), -1, 0, 1, 5, 7, 8, 64, 65, (1 << 31) - 1]


def test_sequences_stay_inside_the_call_whatever_the_device_holds():
    o = (ctypes.c_int * 4)()
    for s, e, n, mq in itertools.product(EDGES, EDGES, EDGES, (0, 5, 7)):
        lib().seq(s, e, n, I64(7), I64(mq), I64(64), o)
        row0, rows, length, bad = list(o)
        assert 0 <= row0 <= 7 and 0 <= rows and row0 + rows <= 7
        right = 0 <= s <= e <= 7 and 0 <= n <= 64 and e - s <= n and e - s <= mq
        assert bad == (not right)
        assert length == (n if right else 0)


def test_pages_stay_inside_the_cache():
    for p in EDGES:
        bad = ctypes.c_int(0)
        r = lib().page(p, 8, ctypes.byref(bad))
        assert 0 <= r < 8 and bool(bad.value) == (not 0 <= p < 8)
        bad = ctypes.c_int(1)  # stays set
        lib().page(3, 8, ctypes.byref(bad))
        assert bad.value == 1


def test_python_descriptions_refuse_before_any_device_call():
    kw = dict(num_pages=1, page_size=16, kv_heads=1, head_size=64)
    with pytest.raises(NotImplementedError, match="type"):
        paged.PagedCache(0, 0, "e4m3", **kw)
    with pytest.raises(ValueError, match="strides"):
        paged.PagedCache(0, 0, "f16", strides=(1, 2), **kw)


def test_null_context_is_an_argument_error():
    so = _lib.load()
    assert so.mmnb_paged_append_dev(None, None, None, None, 0, 0, None, 0, None, 0, None, None, 0,
                                    0, 0, 0, None, 0) == ARG
    assert so.mmnb_paged_attention_dev(None, None, None, None, None, 0, 0, None, 0) == ARG
    assert so.mmnb_paged_attention_shared_dev(None, None, None, None, 0, None, None, 0, 0, None,
                                              0) == ARG
    assert b"null context" in so.mmnb_last_error()
