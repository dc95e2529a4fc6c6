"""Caches whose rows lie as far apart as a tile's loads reach, and farther (a wave per row)."""
import ctypes

import numpy as np
import pytest

from onnx_runtime_dart_amd import _lib, paged
from tests.paged_cases import Case, close
from tests.test_gpu_paged_append import tables, want as appended
from tests.test_gpu_paged_paths import dense

pytestmark = pytest.mark.gpu

TYPES = ["f16", "bf16", "f32"]
FAR = [1 << 23, (1 << 23) + 8]  # elements from row to row


class Spread:
    """The case's cache with row r of all pages, keys then values, r * far elements on."""

    def __init__(self, c, far):
        self.c, self.far = c, far
        self.rows = [np.concatenate([x[:, :, r].ravel() for x in (c.k_raw, c.v_raw)])
                     for r in range(c.page)]
        n, size = c.k_raw[:, :, 0].size, c.k_raw.itemsize
        self.buf = c.ctx.alloc((far * (c.page - 1) + 2 * n) * size)
        c.keep.append(self.buf)
        self.size, at = size, self.buf.ptr.value
        for r, x in enumerate(self.rows):
            self.copy(c.ctx.lib.mmnb_memcpy_h2d, self.at(r), _lib.ptr(x), x.nbytes)
        self.cache = paged.PagedCache(at, at + n * size, c.t, num_pages=c.num_pages,
                                      page_size=c.page, kv_heads=c.kv_heads, head_size=c.head,
                                      strides=(c.kv_heads * c.head, c.head, far))

    def at(self, r):
        return ctypes.c_void_p(self.buf.ptr.value + r * self.far * self.size)

    def copy(self, f, to, src, n):
        _lib.check(f(self.c.ctx.handle, to, src, n))

    def read(self):
        """(k, v) as the case lays them out."""
        out = np.empty((self.c.page, 2) + self.c.k_raw[:, :, 0].shape, self.c.k_raw.dtype)
        for r in range(self.c.page):
            self.copy(self.c.ctx.lib.mmnb_memcpy_d2h, _lib.ptr(out[r]), self.at(r),
                      out[r].nbytes)
        return out.transpose(1, 2, 3, 0, 4)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("kw", [
    dict(new=[1, 1, 3], kv=[200, 33, 70], page=16), dict(new=[70, 5], kv=[70, 300], page=64),
    dict(new=[1, 2], kv=[9, 40], prefix=150, page=16, window=60, two=[3, 0]),
    dict(new=[40, 1], kv=[90, 40], prefix=50, page=8, cap=9.0, bias=True)])
def test_attention(t, far, kw):
    c = Case(**kw, t=t)
    want, tol = dense(c)
    cache = Spread(c, far).cache
    q, out = c.put(c.q), c.put(np.full_like(c.q, 7.0))
    if c.prefix:
        paged.attention_shared(cache, c.batch(), c.put(c.prefix_pages), c.prefix, q, out,
                               heads=c.heads, scores=c.scores(), ctx=c.ctx)
    else:
        paged.attention(cache, c.batch(), q, out, heads=c.heads, scores=c.scores(), ctx=c.ctx)
    y = out.numpy()
    c.free()
    close(y, want, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("far", FAR)
def test_append(t, far):
    c = Case([1, 9], [70, 9], t=t, page=16)
    H, G, D, T = c.heads, c.kv_heads, c.head, c.tokens
    x = np.random.default_rng(2).standard_normal((T, H + 2 * G, D)).astype(np.float32)
    cos, sin = tables(c.max_kv, 16)
    ins = x[:, :H], x[:, H:H + G], x[:, H + G:]
    s = Spread(c, far)
    q, k, v, out = (c.put(y) for y in ins + (np.zeros((T, H, D), np.float32),))
    paged.append(s.cache, c.batch(), q, k, v, c.put(cos), c.put(sin), out, heads=H,
                 max_pos=c.max_kv, half_rot=16, ctx=c.ctx)
    y, kw, vw = appended(c, ins + (cos, sin))
    assert np.array_equal(out.numpy(), y)
    kn, vn = s.read()
    assert np.array_equal(kn, kw) and np.array_equal(vn, vw)
    c.free()


@pytest.mark.parametrize("t", TYPES)
def test_rows_of_broken_sequences(t):
    c = Case([3, 1, 4, 0], [20, 30, 40, 5], t=t, page=16)
    want, tol = dense(c)
    c.kv_len[1] = 1 << 30
    c.start[4] = 2        # the last sequence, without rows, ends before it begins
    cache = Spread(c, FAR[1]).cache
    q, out = c.put(c.q), c.put(np.full_like(c.q, 7.0))
    paged.attention(cache, c.batch(), q, out, heads=c.heads, ctx=c.ctx)
    y = out.numpy()
    c.free()
    assert np.isnan(y[3]).all()
    keep = np.r_[0:3, 4:8]
    close(y[keep], want[keep], tol[keep])
