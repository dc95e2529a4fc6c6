"""Recorded graphs keep the scratch that they were recorded with when a later call grows it."""
import numpy as np
import pytest
import torch

from onnx_runtime_dart_amd import _lib, ops, paged, synth
from tests.paged_cases import Case

pytestmark = pytest.mark.gpu
MB = 1 << 20


@pytest.fixture
def ctx():
    c = _lib.Context(0)  # one whose scratch nothing has grown
    yield c
    c.close()


def replays(ctx, graph, read, first, grow):
    """Replays after a call that grows the scratch, beside memory that may lie where the old
    buffer lay, and with eager work between."""
    for _ in range(3):
        grow()
        ctx.synchronize()
        junk = [ctx.to_device(np.full(64 * MB, 0xFF, np.uint8)) for _ in range(2)]
        ctx.graph_launch(graph)
        ctx.synchronize()
        assert np.array_equal(read(), first)
        for b in junk:
            assert (b.numpy() == 0xFF).all()
            b.free()


def free_bytes():
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("prefix", [0, 200])
def test_paged_step(ctx, prefix):
    c = Case([1, 1], [600, 600], prefix=prefix, heads=8, kv_heads=2, head=128, page=64)
    c.ctx = ctx
    call = c.device()
    call()
    ctx.synchronize()
    first = c.read().copy()
    ctx.graph_begin()
    call()
    g = ctx.graph_end()

    # 300 tokens behind 4000 keys, 32 heads: 201600 pieces of 520 bytes
    put, n = c.put, 300
    rows, out = (put(np.zeros(n * 32 * 128, np.float32)) for _ in range(2))
    kv = put(np.zeros(32 * 64 * 128, np.int16))
    cache = paged.PagedCache(kv, kv, "f16", num_pages=1, page_size=64, kv_heads=32, head_size=128)
    batch = paged.PagedBatch(put(np.arange(n + 1, dtype=np.int32)), put(np.ones(n, np.int32)),
                             put(np.zeros(n, np.int32)), batch=n, tokens=n, page_cols=1, max_q=1,
                             max_kv=1)
    pre = put(np.zeros(63, np.int32))

    def grow():
        paged.attention_shared(cache, batch, pre, 4000, rows, out, heads=32, ctx=ctx)

    replays(ctx, g, c.read, first, grow)
    before = free_bytes()
    ctx.graph_destroy(g)
    assert free_bytes() - before >= 64 * MB  # the outgrown buffer goes with its graph
    grow()
    call()
    ctx.synchronize()
    assert np.array_equal(c.read(), first)
    c.free()


def test_matmul_nbits(ctx):
    """The prefill GEMM's prepared activations."""
    p = synth.mmnb_problem(96, 512, 512, 32, True, seed=1)
    w = ops.pack_nbits(p.b_q, p.scales, p.zero_points, k=512, n=512, bits=4, block_size=32,
                       ctx=ctx)
    a, y = ctx.to_device(p.a), ctx.to_device(np.zeros((96, 512), np.float32))
    big, out = (ctx.to_device(np.zeros((8192, 512), np.float32)) for _ in range(2))

    def call(x, m, to):
        _lib.check(ctx.lib.mmnb_matmul_nbits_dev(ctx.handle, w.handle, x.ptr, m, to.ptr))

    call(a, 96, y)
    ctx.synchronize()
    first = y.numpy()
    ctx.graph_begin()
    call(a, 96, y)
    g = ctx.graph_end()

    def grow():
        y.upload(np.zeros_like(first))
        call(big, 8192, out)

    replays(ctx, g, y.numpy, first, grow)
    ctx.graph_destroy(g)
    w.free()
    for b in (a, y, big, out):
        b.free()
