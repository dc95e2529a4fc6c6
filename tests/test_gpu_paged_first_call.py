"""A step may be recorded after any first call of attention in a context."""
import numpy as np
import pytest

from onnx_runtime_dart_amd import _lib
from tests.paged_cases import Case, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [dict(new=[40], kv=[40], head=64),           # one part
                                   dict(new=[1], kv=[30], head=64),            # whole in a wave
                                   dict(new=[1], kv=[30], head=64, prefix=40)])
def test_a_step_recorded_after_one_call(first):
    ctx = _lib.Context(0)
    warm = Case(**first)
    warm.ctx = ctx
    other = warm.device()
    other()
    c = Case([1, 1], [600, 90], heads=8, kv_heads=2, head=128, page=64)
    c.ctx = ctx
    call = c.device()
    ctx.synchronize()
    ctx.graph_begin()
    call()
    g = ctx.graph_end()
    want, tol = c.want()
    for _ in range(3):
        c.out.upload(np.full(c.out.shape, 7.0, np.float32))
        ctx.graph_launch(g)
        ctx.synchronize()
        close(c.read(), want, tol)
        other()  # eager work between the replays
    ctx.graph_destroy(g)
    warm.free()
    c.free()
    ctx.close()
