"""Attention over a paged cache on the GPU against the 64-bit definition."""
import ctypes

import numpy as np
import pytest

from onnx_runtime_dart_amd import _lib, paged
from oracle import paged as ref
from tests.paged_cases import Case, close, to_type

pytestmark = pytest.mark.gpu

TYPES = ["f16", "bf16", "f32"]
RAGGED = dict(new=[1, 1, 1, 1], kv=[1, 63, 64, 130])
MODS = {
    "plain": {}, "cap": dict(cap=5.0), "window": dict(window=17), "bias": dict(bias=True),
    "two_way": dict(two=[0, 9, 200, 70]), "scale": dict(scale=0.3),
    "all": dict(cap=20.0, window=33, bias=True, two=[1, 0, 5, 140], scale=0.2),
}


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mod", sorted(MODS))
def test_tokens(t, mod):
    Case(**RAGGED, t=t, **MODS[mod]).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mod", sorted(MODS))
def test_prompts(t, mod):
    Case([70, 5, 1, 33], [70, 140, 1, 97], t=t, **MODS[mod]).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv_heads,head", [
    (1, 1, 8), (2, 1, 40), (3, 3, 96), (5, 1, 128), (6, 2, 104), (16, 1, 128), (17, 1, 64),
    (14, 2, 72), (40, 8, 128)])
def test_head_layouts(t, heads, kv_heads, head):
    kw = dict(t=t, heads=heads, kv_heads=kv_heads, head=head)
    Case([1, 1, 1], [5, 200, 77], **kw).check()
    Case([40, 3], [41, 133], **kw).check()


@pytest.mark.parametrize("page", [1, 2, 8, 64, 256])
def test_pages(page):
    Case([1, 1, 9], [300, 1, 131], page=page, t="bf16").check()
    Case([150, 64], [300, 64], page=page, t="f16").check()


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128,
                               129, 255, 257])
def test_rows_of_every_number(n):
    Case([n], [n], t="f16").check()
    Case([n, 1], [n + 100, 3], t="bf16", head=128, heads=8).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kv", [511, 4096, 20011])
def test_long(t, kv):
    Case([1], [kv], t=t, heads=8, kv_heads=2, head=128, page=64).check()
    Case([1, 2], [kv, 700], t=t, heads=4, kv_heads=2, head=128, page=16, cap=9.0).check()


@pytest.mark.parametrize("t", TYPES)
def test_few_rows_far_into_a_long_cache(t):
    Case([40], [9001], t=t, heads=4, kv_heads=1, head=128, page=64).check()
    Case([33, 1], [5000, 6000], t=t, heads=2, kv_heads=2, head=64, page=64, window=1000,
         two=[30, 2500]).check()


@pytest.mark.parametrize("t", TYPES)
def test_longer_prompt(t):
    Case([600], [1111], t=t, heads=4, kv_heads=2, head=128, page=64).check()
    Case([512, 3, 260], [512, 600, 260], t=t, heads=3, kv_heads=1, head=80, page=16,
         window=100).check()


@pytest.mark.parametrize("layout,q_gap,q_off,out_gap", [
    ("apart", 0, 0, 0), ("ghpd", 7, 1, 3), ("apart", 64, 2, 64), ("ghpd", 1, 3, 1)])
@pytest.mark.parametrize("t", TYPES)
def test_strides_and_alignment(t, layout, q_gap, q_off, out_gap):
    kw = dict(t=t, layout=layout, q_gap=q_gap, q_off=q_off, out_gap=out_gap)
    Case([1, 1], [100, 9], **kw).check()
    Case([50, 20], [100, 33], **kw).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf])
def test_what_no_row_sees_does_not_reach_it(t, poison):
    Case([1, 1], [130, 5], t=t, poison=poison).check()
    Case([90, 4], [130, 33], t=t, poison=poison).check()
    Case([1, 3], [30, 5], t=t, poison=poison, prefix=77).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new,kv,window", [([1], [200], 64), ([100], [200], 0), ([100], [200], 20),
                                           ([3], [400], 0)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf, 60000.0])
def test_keys_and_values_that_only_some_rows_see(t, new, kv, window, what):
    """A key of NaN or infinity reaches the rows that see it, and those alone."""
    for at in (2, 130, 190, 199):
        for which in ("k", "v"):
            c = Case(new, kv, t=t, window=window, heads=4, kv_heads=2, head=64)
            page = c.pages[0, at // c.page]
            raw, val = to_type(np.full(8, what), t)
            getattr(c, which + "_raw")[page, 1, at % c.page, 8:16] = raw
            getattr(c, which)[page, 1, at % c.page, 8:16] = val
            c.check()


@pytest.mark.parametrize("t", TYPES)
def test_queries_of_nan_and_infinity_stay_in_their_rows(t):
    for new, kv in (([1, 1, 1], [40, 50, 300]), ([60, 9, 2], [60, 50, 300])):
        c = Case(new, kv, t=t)
        c.q[1, 2, 5] = np.nan
        c.q[0, 1] = 0.0
        c.check()


@pytest.mark.parametrize("t", TYPES)
def test_large_and_small_queries(t):
    """Rows of far apart sizes, values up to where a score leaves binary32's range."""
    for new, kv in (([1] * 6, [90] * 6), ([6, 64], [90, 64])):
        c = Case(new, kv, t=t)
        for i, size in enumerate([1e-30, 1e-12, 1e-4, 1.0, 30.0, 1e4]):
            c.q[i] *= np.float32(size)
        c.check()


@pytest.mark.parametrize("t", TYPES)
def test_rows_that_see_nothing_are_zero(t):
    # every row sees its own key: only scores of -infinity leave it nothing
    y = Case([0, 2, 0, 1], [0, 2, 50, 1], t=t).check()
    assert np.isfinite(y).all()
    c = Case([1, 2], [10, 20], t=t)
    c.k_raw[:] = to_type(np.full(c.k.shape, -np.inf), t)[0]
    c.k[:] = -np.inf
    c.q[:] = 1.0
    assert (c.check() == 0).all()


def test_empty_calls():
    Case([], []).device()()
    Case([0, 0], [5, 0]).device()()
    _lib.default_context().synchronize()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new,kv", [([1, 1, 1, 1], [90, 200, 20, 40]),
                                    ([40, 90, 3, 30], [90, 200, 20, 40])])
def test_page_numbers_outside_the_cache(t, new, kv):
    """They are never followed: the rows that see a key of such a page become NaN."""
    for bad in (-1, 1 << 30, -(1 << 31)):
        c = Case(new, kv, t=t)
        lost = 7  # of sequence 1: keys 112 ..
        c.pages[1, lost] = bad
        y = c.run()
        c.pages[1, lost] = 0
        want, tol = c.want()
        c.free()
        for b, row, own in ref.rows(c.start, c.kv_len):
            if b == 1 and own >= lost * c.page:
                assert np.isnan(y[row]).all()
            else:
                close(y[row], want[row], tol[row])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new,kv", [([1, 1, 1, 1], [90, 200, 20, 40]),
                                    ([40, 90, 3, 30], [90, 200, 20, 40])])
def test_lengths_that_break_the_promises(t, new, kv):
    """Such a sequence's rows become NaN, the others are as ever."""
    for wrong in (-5, 1 << 30, 201, 0):
        c = Case(new, kv, t=t)
        call = c.device()
        lens = c.kv_len.copy()
        lens[1] = wrong
        for buf in c.keep:
            if buf.shape == c.kv_len.shape and buf.dtype == np.int32 and \
                    np.array_equal(buf.numpy(), c.kv_len):
                buf.upload(lens)
        call()
        c.ctx.synchronize()
        y = c.read()
        want, tol = c.want()
        c.free()
        for b, row, _ in ref.rows(c.start, c.kv_len):
            if b == 1:
                assert np.isnan(y[row]).all()
            else:
                close(y[row], want[row], tol[row])


def test_row_starts_that_break_the_promises():
    c = Case([2, 3, 4], [20, 30, 40], max_q=3)
    y = c.run()
    want, tol = c.want()
    c.free()
    close(y[:5], want[:5], tol[:5])
    assert np.isnan(y[5:]).all()
    c = Case([2, 3, 4], [20, 30, 40])
    c.start[:] = [0, 2, 500, 9]
    y = c.run()
    c.free()
    close(y[:2], want[:2], tol[:2])
    assert np.isnan(y[2:9]).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("prefix", [1, 15, 16, 300, 1000])
@pytest.mark.parametrize("mod", ["plain", "all", "window"])
def test_shared_prefix(t, prefix, mod):
    Case(**RAGGED, t=t, prefix=prefix, head=128, **MODS[mod]).check()
    Case([20, 1, 7, 3], [20, 1, 60, 33], t=t, prefix=prefix, **MODS[mod]).check()


@pytest.mark.parametrize("t", TYPES)
def test_shared_prefix_of_many(t):
    Case([1] * 70, [1 + 3 * i for i in range(70)], t=t, prefix=2000, heads=8, kv_heads=2,
         head=128, page=64, seed=3).check()
    Case([1] * 9, [1] * 9, t=t, prefix=777, heads=7, kv_heads=7, head=64, page=8).check()


def test_shared_prefix_with_a_bad_page():
    c = Case([1, 2], [5, 20], prefix=100)
    c.prefix_pages[3] = 1 << 20
    assert np.isnan(c.run()).all()
    c.free()


@pytest.mark.parametrize("t", TYPES)
def test_same_bits_every_time(t):
    for kw in (dict(new=[1, 1], kv=[3000, 50]), dict(new=[90, 3], kv=[300, 3]),
               dict(new=[1, 1], kv=[30, 50], prefix=999)):
        c = Case(**kw, t=t, heads=8, head=128)
        call = c.device()
        got = []
        for _ in range(4):
            call()
            c.ctx.synchronize()
            got.append(c.read().copy())
        c.free()
        for y in got[1:]:
            assert np.array_equal(y.view(np.int32), got[0].view(np.int32))


@pytest.mark.parametrize("prefix", [0, 200])
def test_captured_step_follows_the_lengths(prefix):
    """A recorded call replayed while the sequences grow under it, up to max_kv."""
    c = Case([1, 1], [600, 600], prefix=prefix, heads=8, kv_heads=2, head=128, page=64)
    call = c.device()
    call()
    c.ctx.synchronize()
    lens = [b for b in c.keep if b.shape == (2,) and b.dtype == np.int32 and
            np.array_equal(b.numpy(), c.kv_len)][0]
    c.ctx.graph_begin()
    call()
    g = c.ctx.graph_end()
    for step in ([1, 2], [64, 65], [300, 7], [600, 599], [5, 600]):
        lens.upload(np.array(step, np.int32))
        c.kv_len = np.array(step, np.int32)
        c.ctx.synchronize()
        c.ctx.graph_launch(g)
        c.ctx.synchronize()
        y = c.read()
        want, tol = c.want()
        close(y, want, tol)
        call()  # eager work between the replays
        c.ctx.synchronize()
        assert np.array_equal(c.read(), y)
    c.ctx.graph_destroy(g)
    c.free()


def test_offsets_past_32_bits():
    """Pages that lie beyond 2^32 bytes and 2^31 elements of the cache."""
    c = Case([1, 30], [200, 100], t="f16", heads=2, kv_heads=1, head=64, page=64, spare=5)
    span = 1 << 28  # elements from page to page
    lib, ctx = c.ctx.lib, c.ctx
    bufs = [ctx.alloc(2 * (span * (c.num_pages - 1) + c.page * c.head)) for _ in range(2)]
    for buf, raw in zip(bufs, (c.k_raw, c.v_raw)):
        for i in range(c.num_pages):
            x = np.ascontiguousarray(raw[i])
            _lib.check(lib.mmnb_memcpy_h2d(ctx.handle, ctypes.c_void_p(buf.ptr.value +
                                                                       2 * span * i),
                                           _lib.ptr(x), x.nbytes))
    cache = paged.PagedCache(bufs[0], bufs[1], "f16", num_pages=c.num_pages, page_size=64,
                             kv_heads=1, head_size=64, strides=(span, 64 * 64, 64))
    assert span * (c.num_pages - 1) > 1 << 31
    q, out = c.put(c.q), c.put(np.zeros_like(c.q))
    paged.attention(cache, c.batch(), q, out, heads=2, ctx=ctx)
    y = out.numpy()
    want, tol = c.want()
    close(y, want, tol)
    for b in bufs:
        b.free()
    c.free()
