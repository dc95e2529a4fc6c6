"""Which scratch buffers recorded graphs keep, on the CPU (csrc/mmnb_graphs.h built for the
host)."""
import ctypes
import functools
import shutil
import subprocess
import tempfile
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "onnx_runtime_dart_amd" / "csrc"
SHIM = """
#include "mmnb_graphs.h"
using namespace mmnb;
typedef void (*Free)(void *);
extern "C" {
void *make() { return new GraphBuffers; }
void drop(void *g) { delete (GraphBuffers *)g; }
void begin(void *g) { ((GraphBuffers *)g)->begin(); }
void take(void *g, int slot, void *p) { ((GraphBuffers *)g)->take(slot, p); }
int end(void *g, void *graph) { return ((GraphBuffers *)g)->end(graph); }
int held(void *g, void *p) { return ((GraphBuffers *)g)->held(p); }
int retire(void *g, void *p) { return ((GraphBuffers *)g)->retire(p); }
void destroyed(void *g, void *graph, Free f) { ((GraphBuffers *)g)->destroyed(graph, f); }
void clear(void *g, Free f) { ((GraphBuffers *)g)->clear(f); }
}
"""
FREE = ctypes.CFUNCTYPE(None, ctypes.c_void_p)


@functools.lru_cache(None)
def lib():
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = Path(tempfile.mkdtemp())
    (d / "graphs.cpp").write_text(SHIM)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-O1", "-shared", "-fPIC", "-I",
                    str(CSRC), str(d / "graphs.cpp"), "-o", str(d / "graphs.so")], check=True)
    so = ctypes.CDLL(str(d / "graphs.so"))
    so.make.restype = ctypes.c_void_p
    return so


class Buffers:
    def __init__(self):
        self.h, self.freed = ctypes.c_void_p(lib().make()), []
        self.cb = FREE(lambda p: self.freed.append(p))

    def __getattr__(self, name):
        def call(*args):
            args = [ctypes.c_void_p(a) if i or name not in ("take",) else a
                    for i, a in enumerate(args)]
            if name in ("destroyed", "clear"):
                args.append(self.cb)
            return getattr(lib(), name)(self.h, *args)
        return call

    def record(self, graph, *buffers):
        self.begin()
        for slot, p in buffers:
            self.take(slot, p)
        assert self.end(graph)


def test_an_outgrown_buffer_lives_as_long_as_a_graph_that_holds_it():
    b = Buffers()
    b.record(1, (11, 100), (2, 50))
    b.record(2, (11, 100))
    assert b.held(100) and b.held(50) and not b.held(200)
    assert b.retire(100)
    b.destroyed(1)
    assert b.freed == [] and b.held(100) and not b.held(50)
    b.destroyed(2)
    assert b.freed == [100] and not b.held(100)
    b.destroyed(2)
    assert b.freed == [100]


def test_a_buffer_that_is_still_the_contexts_is_not_freed_with_the_graph():
    b = Buffers()
    b.record(1, (3, 10))
    b.destroyed(1)
    assert b.freed == [] and not b.held(10)


def test_several_growths_keep_one_buffer_for_each_graph():
    b = Buffers()
    for i in range(5):
        b.record(i + 1, (11, 1000 + i))
        assert b.retire(1000 + i)
    for i in (2, 0, 4, 1, 3):
        b.destroyed(i + 1)
        assert b.freed[-1] == 1000 + i
    assert len(b.freed) == 5


def test_a_recording_given_up_holds_nothing():
    b = Buffers()
    b.begin()
    b.take(11, 77)
    b.begin()  # the next one
    assert b.end(1) and not b.held(77)
    assert not b.held(None)


def test_the_context_frees_what_is_left():
    b = Buffers()
    b.record(1, (11, 5))
    b.record(2, (11, 6))
    b.retire(5), b.retire(6)
    b.clear()
    assert sorted(b.freed) == [5, 6]
