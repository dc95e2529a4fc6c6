"""Device state of a paged batch and its 64-bit result, for the GPU tests."""
import numpy as np
import torch

from onnx_runtime_dart_amd import _lib, paged
from oracle import paged as ref

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# bits to which queries and softmax weights are held on the way into the matrix cores
SPLIT_BITS = {"f32": 24, "f16": 22, "bf16": 24}


def to_type(x, t):
    """x (float array) rounded to the cache's type: (its bytes' array, its float64 values)."""
    y = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[t])
    raw = y.numpy() if t == "f32" else y.view(torch.int16).numpy()
    return raw, y.double().numpy()


class Case:
    """A batch of sequences with `new` rows and `kv` keys each."""

    def __init__(self, new, kv, *, heads=4, kv_heads=2, head=64, t="f16", page=16, seed=0,
                 prefix=0, cap=0.0, window=0, bias=False, two=None, scale=0.0, layout="ghpd",
                 spare=3, poison=None, max_q=None, max_kv=None, q_gap=0, q_off=0, out_gap=0):
        rng = np.random.default_rng(seed)
        self.ctx = _lib.default_context()
        self.t, self.heads, self.kv_heads, self.head, self.page = t, heads, kv_heads, head, page
        self.new, self.kv = list(new), list(kv)
        self.tokens, self.prefix = sum(new), prefix
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.kv_len = np.array(kv, np.int32)
        need = [-(-n // page) for n in kv]
        pre = -(-prefix // page)
        self.cols = max(need + [1])
        self.num_pages = sum(need) + pre + spare
        order = rng.permutation(self.num_pages).astype(np.int32)
        self.prefix_pages = order[:pre]
        self.pages = np.full((len(kv), self.cols), -1, np.int32)
        at = pre
        for b, n in enumerate(need):
            self.pages[b, :n] = order[at:at + n]
            at += n
        shape = (self.num_pages, kv_heads, page, head)
        big = np.ones(head)
        big[rng.permutation(head)[:max(1, head // 32)]] = 4.0
        k, v = rng.standard_normal(shape) * big, rng.standard_normal(shape)
        if poison is not None:  # what no key of a sequence lies in
            used = np.zeros(shape[:1] + shape[2:3], bool)
            for pages, n in [(self.prefix_pages, prefix)] + list(zip(self.pages, kv)):
                j = np.arange(n)
                used[pages[j // page], j % page] = True
            k = np.where(used[:, None, :, None], k, poison)
            v = np.where(used[:, None, :, None], v, poison)
        self.k_raw, self.k = to_type(k, t)
        self.v_raw, self.v = to_type(v, t)
        self.layout = layout
        self.q = (rng.standard_normal((self.tokens, heads, head)) * 1.5).astype(np.float32)
        self.q_gap, self.q_off, self.out_gap = q_gap, q_off, out_gap
        self.slopes = (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32) \
            if bias else None
        self.two = None if two is None else np.array(two, np.int32)
        self.cap, self.window, self.scale = cap, window, scale
        self.max_q = max(self.new + [0]) if max_q is None else max_q
        self.max_kv = max(self.kv + [0]) if max_kv is None else max_kv
        self.keep = []

    def put(self, x):
        buf = self.ctx.to_device(np.ascontiguousarray(x))
        self.keep.append(buf)
        return buf

    def cache(self):
        """The cache on the device in the case's layout."""
        if self.layout == "ghpd":      # [pages, kv_heads, page, head], the default
            kd, vd, strides = self.put(self.k_raw), self.put(self.v_raw), None
            k, v = kd.ptr.value, vd.ptr.value
        else:                          # [pages, page, 2 (k, v), kv_heads, head + 8]
            both = np.stack([self.k_raw, self.v_raw], 0).transpose(1, 3, 0, 2, 4)
            both = np.pad(both, [(0, 0)] * 4 + [(0, 8)])
            kd = self.put(both)
            w = self.head + 8
            strides = (self.page * 2 * self.kv_heads * w, w, 2 * self.kv_heads * w)
            k = kd.ptr.value
            v = k + self.kv_heads * w * both.itemsize
        return paged.PagedCache(k, v, self.t, num_pages=self.num_pages, page_size=self.page,
                                kv_heads=self.kv_heads, head_size=self.head, strides=strides)

    def batch(self):
        return paged.PagedBatch(self.put(self.start), self.put(self.kv_len),
                                self.put(self.pages), batch=len(self.kv), tokens=self.tokens,
                                page_cols=self.cols, max_q=self.max_q, max_kv=self.max_kv)

    def scores(self):
        return paged.Scores(self.scale, self.cap, self.window,
                            None if self.slopes is None else self.put(self.slopes),
                            None if self.two is None else self.put(self.two))

    def device(self):
        """Puts everything on the device; returns call() and read()."""
        w = self.heads * self.head
        ldq, ldo = w + self.q_gap, w + self.out_gap
        q = np.full(self.tokens * ldq + self.q_off, np.nan, np.float32)
        q[self.q_off:].reshape(self.tokens, ldq)[:, :w] = self.q.reshape(self.tokens, w)
        qd = self.put(q)
        self.out = self.put(np.full((self.tokens, ldo), 7.0, np.float32))
        cache, batch, scores = self.cache(), self.batch(), self.scores()
        if self.prefix:
            pre = self.put(self.prefix_pages)
            return lambda: paged.attention_shared(
                cache, batch, pre, self.prefix, qd.ptr.value + 4 * self.q_off, self.out,
                heads=self.heads, scores=scores, ldq=ldq, ldo=ldo, ctx=self.ctx)
        return lambda: paged.attention(cache, batch, qd.ptr.value + 4 * self.q_off, self.out,
                                       heads=self.heads, scores=scores, ldq=ldq, ldo=ldo,
                                       ctx=self.ctx)

    def read(self):
        w = self.heads * self.head
        y = self.out.numpy()
        assert (y[:, w:] == 7.0).all()
        return y[:, :w].reshape(self.tokens, self.heads, self.head)

    def run(self):
        self.device()()
        self.ctx.synchronize()
        return self.read()

    def want(self):
        return ref.attend(self.q, self.k, self.v, self.start, self.kv_len, self.pages,
                          prefix_pages=self.prefix_pages, prefix=self.prefix, scale=self.scale,
                          cap=self.cap, window=self.window, slopes=self.slopes, two=self.two,
                          split_bits=SPLIT_BITS[self.t])

    def free(self):
        for b in self.keep:
            b.free()
        self.keep = []

    def check(self):
        y = self.run()
        want, tol = self.want()
        self.free()
        close(y, want, tol)
        return y


def close(y, want, tol):
    """y within tol of want, and not finite exactly where want is not."""
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(y), np.isnan(want))
    assert np.array_equal(np.isfinite(y), fine)
    assert np.array_equal(np.sign(y[~fine & ~np.isnan(y)]), np.sign(want[~fine & ~np.isnan(want)]))
    off = np.abs(y.astype(np.float64) - want)[fine]
    worst = float((off / tol[fine]).max()) if off.size else 0.0
    print(f"largest error {off.max() if off.size else 0:.3g}, {worst:.3g} of the tolerance",
          flush=True)
    assert worst <= 1.0, worst
