"""The factors of a score, on the CPU (csrc/mmnb_paged_plan.h built for the host)."""
import ctypes
import functools
import math
import shutil
import subprocess
import tempfile
from pathlib import Path

import numpy as np
import pytest

from onnx_runtime_dart_amd import _lib

CSRC = Path(__file__).resolve().parents[1] / "onnx_runtime_dart_amd" / "csrc"
SHIM = """
#include "mmnb_paged_plan.h"
extern "C" int factors(const mmnb_paged_scores *s, int64_t head, float *o) {
  const mmnb::PagedFactors f = mmnb::paged_factors(s, head);
  o[0] = f.mul, o[1] = f.in_mul;
  return f.capped;
}
"""
TINY, HUGE = 1e-45, 3.4028234e38


@functools.lru_cache(None)
def lib():
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = Path(tempfile.mkdtemp())
    (d / "f.cpp").write_text(SHIM)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-O1", "-shared", "-fPIC", "-I",
                    str(CSRC), str(d / "f.cpp"), "-o", str(d / "f.so")], check=True)
    return ctypes.CDLL(str(d / "f.so"))


def factors(scale, cap, head=64):
    o = (ctypes.c_float * 2)()
    s = _lib.PagedScores(scale, cap, 0, None, None)
    capped = lib().factors(ctypes.byref(s), ctypes.c_int64(head), o)
    return bool(capped), float(o[0]), float(o[1])


@pytest.mark.parametrize("scale", [0.0, TINY, 1e-30, 0.1, 1e30, HUGE])
@pytest.mark.parametrize("cap", [0.0, TINY, 1e-40, 1e-30, 1.0, 50.0, 1e20, 2.0 ** 100, 1.3e30, 1e35,
                                 HUGE])
def test_factors_are_finite_and_the_formulas(scale, cap):
    capped, mul, in_mul = factors(scale, cap)
    assert math.isfinite(mul) and math.isfinite(in_mul)
    assert capped == (0 < np.float32(cap) <= 2.0 ** 100)
    s = float(np.float32(scale)) if np.float32(scale) > 0 else 0.125
    want = float(np.float32(cap)) if capped else s
    if TINY < want < 2e38:  # one rounding; below the normal numbers half a step of 2^-149
        assert abs(mul - want * math.log2(math.e)) <= max(2.0 ** -24 * mul, 2.0 ** -150)
    ratio = s / want if capped else 0.0
    if ratio < HUGE:
        assert abs(in_mul - ratio) <= max(2.0 ** -24 * ratio, 2.0 ** -150)


def test_default_scale():
    o = (ctypes.c_float * 2)()
    assert lib().factors(None, ctypes.c_int64(96), o) == 0
    assert o[0] == np.float32(float(np.float32(1 / math.sqrt(96))) * math.log2(math.e))
