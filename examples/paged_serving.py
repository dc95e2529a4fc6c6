"""An int4 attention layer that serves several talks from one paged key/value cache.

    python examples/paged_serving.py [--talks 6] [--steps 16] [--type f16]

All talks begin with the same system prompt, which the cache holds once.  Each step projects the
talks' rows to queries, keys and values (MatMulNBits), stores the keys and values in their pages
with the rotary embedding (paged.append), attends behind the shared prompt
(paged.attention_shared) and projects back.  Prompts of uneven length run as one ragged batch;
the steps of single tokens replay one recorded graph, whose lengths and page tables are device
memory that is uploaded between the steps.
"""
import argparse
import sys
import time
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from onnx_runtime_dart_amd import _lib, ops, paged, synth  # noqa: E402


class Pages:
    """The cache's free pages and every talk's page table."""

    def __init__(self, num_pages, page_size, seed=0):
        self.size = page_size
        self.free = list(np.random.default_rng(seed).permutation(num_pages))
        self.tables = {}

    def grow(self, talk, length):
        """Gives the talk pages for `length` keys."""
        t = self.tables.setdefault(talk, [])
        while len(t) * self.size < length:
            t.append(int(self.free.pop()))

    def table(self, talks, cols):
        out = np.zeros((len(talks), cols), np.int32)
        for i, talk in enumerate(talks):
            out[i, :len(self.tables[talk])] = self.tables[talk]
        return out


class Layer:
    """y = x + W_o attention(W_qkv x)."""

    def __init__(self, ctx, *, hidden=512, heads=8, kv_heads=2, head=64, block=32, max_pos=4096,
                 num_pages=256, page=16, dtype="f16", seed=0):
        self.ctx, self.hidden, self.heads, self.kv_heads, self.head = ctx, hidden, heads, \
            kv_heads, head
        self.width, self.max_pos = (heads + 2 * kv_heads) * head, max_pos
        self.weights = [synth.mmnb_weights(k, n, block, True, seed + i, (0.002, 0.006))
                        for i, (k, n) in enumerate([(hidden, self.width),
                                                    (heads * head, hidden)])]
        self.qkv, self.proj = (
            ops.pack_nbits(b, s, z, k=k, n=n, bits=4, block_size=block, ctx=ctx)
            for (b, s, z), (k, n) in zip(self.weights, [(hidden, self.width),
                                                        (heads * head, hidden)]))
        self.half = head // 2
        angle = np.outer(np.arange(max_pos), 1e4 ** (-np.arange(self.half) / self.half))
        self.tables = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.cos, self.sin = (ctx.to_device(t) for t in self.tables)
        size = num_pages * kv_heads * page * head * (4 if dtype == "f32" else 2)
        self.k, self.v = ctx.alloc(size), ctx.alloc(size)
        self.cache = paged.PagedCache(self.k, self.v, dtype, num_pages=num_pages, page_size=page,
                                      kv_heads=kv_heads, head_size=head)
        self.pages = Pages(num_pages, page, seed)

    def buffers(self, rows):
        f = self.ctx.to_device
        return {"x": f(np.zeros((rows, self.hidden), np.float32)),
                "qkv": f(np.zeros((rows, self.width), np.float32)),
                "q": f(np.zeros((rows, self.heads * self.head), np.float32)),
                "o": f(np.zeros((rows, self.heads * self.head), np.float32)),
                "y": f(np.zeros((rows, self.hidden), np.float32))}

    def run(self, buf, batch, rows, prefix_pages=None, prefix=0):
        """One pass over the rows in buf["x"]; nothing waits for the device."""
        lib, c = self.ctx.lib, self.ctx.handle
        _lib.check(lib.mmnb_matmul_nbits_dev(c, self.qkv.handle, buf["x"].ptr, rows,
                                             buf["qkv"].ptr))
        at, D = buf["qkv"].ptr.value, self.head
        paged.append(self.cache, batch, at, at + 4 * self.heads * D,
                     at + 4 * (self.heads + self.kv_heads) * D, self.cos, self.sin, buf["q"],
                     heads=self.heads, max_pos=self.max_pos, half_rot=self.half,
                     first_pos=prefix, ldq=self.width, ldk=self.width, ldv=self.width,
                     ctx=self.ctx)
        if prefix:
            paged.attention_shared(self.cache, batch, prefix_pages, prefix, buf["q"], buf["o"],
                                   heads=self.heads, ctx=self.ctx)
        else:
            paged.attention(self.cache, batch, buf["q"], buf["o"], heads=self.heads,
                            ctx=self.ctx)
        _lib.check(lib.mmnb_matmul_nbits_dev(c, self.proj.handle, buf["o"].ptr, rows,
                                             buf["y"].ptr))


def serve(layer, system, prompts, steps):
    """system [n, hidden] and prompts (a list of [m, hidden]) are hidden rows.  Every talk's next
    row is its last one's result; returns the rows of each talk, results first to last."""
    ctx, pages, n = layer.ctx, layer.pages, len(prompts)

    def batch(talks, new, length, cols, max_q, max_kv):
        start = ctx.to_device(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        lens = ctx.to_device(np.array(length, np.int32))
        table = ctx.to_device(pages.table(talks, cols))
        return lens, table, paged.PagedBatch(start, lens, table, batch=len(talks),
                                             tokens=int(sum(new)), page_cols=cols, max_q=max_q,
                                             max_kv=max_kv)

    # the system prompt, once: its pages are the prefix of every talk
    pages.grow("system", len(system))
    buf = layer.buffers(len(system))
    buf["x"].upload(system)
    cols = len(pages.tables["system"])
    _, prefix_pages, b = batch(["system"], [len(system)], [len(system)], cols, len(system),
                               len(system))
    layer.run(buf, b, len(system))

    # the talks' own prompts, one ragged batch
    lens = [len(p) for p in prompts]
    most = max(lens) + steps
    cols = -(-most // pages.size)
    for i, m in enumerate(lens):
        pages.grow(i, m + steps)
    buf = layer.buffers(sum(lens))
    buf["x"].upload(np.concatenate(prompts))
    _, _, b = batch(range(n), lens, lens, cols, max(lens), most)
    layer.run(buf, b, sum(lens), prefix_pages, len(system))
    y = buf["y"].numpy() + np.concatenate(prompts)
    ends = np.cumsum(lens)
    out = [[y[e - m:e]] for e, m in zip(ends, lens)]

    # single tokens: the pass is recorded once and replayed
    buf = layer.buffers(n)
    dev_lens, _, b = batch(range(n), [1] * n, lens, cols, 1, most)
    graph = None
    for _ in range(steps):
        x = np.stack([o[-1][-1] for o in out])
        lens = [m + 1 for m in lens]
        buf["x"].upload(x)
        dev_lens.upload(np.array(lens, np.int32))
        if graph is None:
            layer.run(buf, b, n, prefix_pages, len(system))
            ctx.synchronize()
            ctx.graph_begin()
            layer.run(buf, b, n, prefix_pages, len(system))
            graph = ctx.graph_end()
        else:
            ctx.graph_launch(graph)
        y = buf["y"].numpy() + x
        for o, row in zip(out, y):
            o.append(row[None])
    if graph is not None:
        ctx.graph_destroy(graph)
    return [np.concatenate(o) for o in out]


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--talks", type=int, default=6)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--type", default="f16", choices=["f16", "bf16", "f32"])
    a = ap.parse_args()
    layer = Layer(_lib.default_context(), dtype=a.type)
    rng = np.random.default_rng(1)
    system = rng.standard_normal((200, layer.hidden)).astype(np.float32)
    prompts = [rng.standard_normal((5 + 13 * i, layer.hidden)).astype(np.float32)
               for i in range(a.talks)]
    t = time.time()
    out = serve(layer, system, prompts, a.steps)
    print(f"{a.talks} talks of {[len(o) for o in out]} rows behind {len(system)} shared ones in "
          f"{time.time() - t:.3f} s; last row's first values: {out[-1][-1, :4]}")


if __name__ == "__main__":
    main()
