"""Storing rows in a paged cache on the GPU: the same bits as the definition."""
import numpy as np
import pytest

from onnx_runtime_dart_amd import _lib, paged
from oracle import paged as ref
from tests.paged_cases import Case, to_type

pytestmark = pytest.mark.gpu

TYPES = ["f16", "bf16", "f32"]


def tables(max_pos, half, seed=0):
    a = np.outer(np.arange(max_pos), 1e4 ** (-np.arange(half) / max(1, half)))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def run(c, half, *, inter=False, first=0, max_pos=None, in_place=False, no_q=False, fused=False):
    """Appends random rows; returns the inputs and what the device holds afterwards."""
    rng = np.random.default_rng(5)
    H, G, D, T = c.heads, c.kv_heads, c.head, c.tokens
    max_pos = first + c.max_kv if max_pos is None else max_pos
    x = rng.standard_normal((T, H + 2 * G, D)).astype(np.float32)
    q, k, v = x[:, :H], x[:, H:H + G], x[:, H + G:]
    cos, sin = tables(max_pos, half)
    cache, batch = c.cache(), c.batch()
    kb, vb = c.keep[0], c.keep[1]
    cd, sd = (c.put(cos), c.put(sin)) if half else (None, None)
    if fused:  # one row of projections, three floats before it
        buf = c.put(np.concatenate([np.zeros(3, np.float32), x.ravel()]))
        at, ld = buf.ptr.value + 12, (H + 2 * G) * D
        qa, ka, va = at, at + 4 * H * D, at + 4 * (H + G) * D
    else:
        qa, ka, va = (c.put(y).ptr.value for y in (q, k, v))
        ld = None
    out = c.put(np.full((T, H, D), 7.0, np.float32))
    oa = qa if in_place else out.ptr.value
    paged.append(cache, batch, None if no_q else qa, ka, va, cd, sd, None if no_q else oa,
                 heads=H, max_pos=max_pos, half_rot=half, interleaved=inter, first_pos=first,
                 ldq=ld, ldk=ld, ldv=ld, ldqo=ld if in_place else None, ctx=c.ctx)
    c.ctx.synchronize()
    if in_place:
        buf = [b for b in c.keep if b.ptr.value <= qa < b.ptr.value + b.nbytes][0]
        y = buf.numpy().ravel()[(qa - buf.ptr.value) // 4:]
        y = y[:T * (ld or H * D)].reshape(T, -1)[:, :H * D].reshape(T, H, D)
    else:
        y = out.numpy()
    if c.layout == "ghpd":
        kn, vn = kb.numpy(), vb.numpy()
    else:
        both = kb.numpy()[..., :D].transpose(2, 0, 3, 1, 4)
        kn, vn = both[0], both[1]
    return (q, k, v, cos, sin), (y, kn, vn)


def want(c, ins, *, inter=False, first=0, skip=()):
    q, k, v, cos, sin = ins
    y, kw, vw = np.full_like(q, 7.0), c.k_raw.copy(), c.v_raw.copy()
    for b, row, own in ref.rows(c.start, c.kv_len):
        if b in skip:
            y[row] = np.nan
            continue
        p = first + own
        if p < len(cos):
            y[row], kr = (ref.rotate(z[row], cos[p], sin[p], inter) for z in (q, k))
        else:
            y[row], kr = (z[row].copy() for z in (q, k))
            y[row][:, :2 * cos.shape[1]] = kr[:, :2 * cos.shape[1]] = np.nan
        page = c.pages[b, own // c.page]
        if 0 <= page < c.num_pages:
            kw[page, :, own % c.page] = to_type(kr, c.t)[0]
            vw[page, :, own % c.page] = to_type(v[row], c.t)[0]
    return y, kw, vw


def same(got, exp, t):
    for x, y in zip(got, exp):
        nx, ny = (z if z.dtype == np.float32 else
                  (z & 0x7fff) > (0x7c00 if t == "f16" else 0x7f80) for z in (x, y))
        if x.dtype == np.float32:
            assert np.array_equal(nx, ny, equal_nan=True)
        else:  # any NaN is a NaN
            assert np.array_equal(nx, ny)
            assert np.array_equal(x[~nx], y[~ny])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("head,half", [(64, 32), (128, 64), (128, 16), (96, 24), (40, 5), (8, 4),
                                       (72, 33), (64, 0), (16, 1)])
def test_rows_and_rotation(t, inter, head, half):
    c = Case([1, 5, 0, 33], [1, 60, 7, 100], t=t, head=head, heads=6, kv_heads=3)
    ins, got = run(c, half, inter=inter)
    same(got, want(c, ins, inter=inter), t)
    c.free()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("half", [32, 7])
@pytest.mark.parametrize("kw", [dict(in_place=True), dict(fused=True), dict(no_q=True),
                                dict(fused=True, in_place=True), dict(first=100)])
def test_forms(t, half, kw):
    c = Case([1, 9], [70, 9], t=t, layout="apart" if kw.get("fused") else "ghpd")
    ins, got = run(c, half, **kw)
    exp = want(c, ins, first=kw.get("first", 0))
    if kw.get("no_q"):
        exp[0][:] = 7.0
    same(got, exp, t)
    c.free()


@pytest.mark.parametrize("t", TYPES)
def test_many_sequences(t):
    n = 300  # more than a workgroup's threads
    c = Case([1 + i % 3 for i in range(n)], [3 + i for i in range(n)], t=t, heads=2, kv_heads=1,
             head=32, page=8)
    ins, got = run(c, 16)
    same(got, want(c, ins), t)
    c.free()


@pytest.mark.parametrize("t", TYPES)
def test_bad_pages_and_positions(t):
    """Rows of a page outside the cache are dropped, positions past the tables are NaN."""
    for bad in (-1, 1 << 30):
        c = Case([40, 3], [64, 20], t=t)
        c.pages[0, 2] = bad
        ins, got = run(c, 32, max_pos=60)
        same(got, want(c, ins), t)
        c.free()


@pytest.mark.parametrize("wrong", [-3, 5, 1 << 30])
def test_bad_lengths_store_nothing(wrong):
    c = Case([4, 9], [40, 60])
    right = c.kv_len
    c.kv_len = np.array([40, wrong], np.int32)
    ins, got = run(c, 32)
    c.kv_len = right
    same(got, want(c, ins, skip=(1,)), "f16")
    c.free()


@pytest.mark.parametrize("t", TYPES)
def test_values_past_the_types_range_and_not_finite(t):
    c = Case([3], [9], t=t)
    rng = np.random.default_rng(0)
    ins, _ = run(c, 0)
    c.free()
    v = np.array(ins[2])
    v.ravel()[:8] = [np.inf, -np.inf, np.nan, 70000.0, -1e38, 1e-8, 6e-8, -0.0]
    c = Case([3], [9], t=t)
    cache, batch = c.cache(), c.batch()
    kb, vb = c.keep[0], c.keep[1]
    paged.append(cache, batch, None, c.put(v), c.put(v), None, None, None, heads=1, max_pos=0,
                 half_rot=0, ctx=c.ctx)
    c.ctx.synchronize()
    with np.errstate(over="ignore"):
        exp = want(c, (np.zeros((3, 1, c.head), np.float32), v, v, np.zeros((9, 0)),
                       np.zeros((9, 0))))
    same((kb.numpy(), vb.numpy()), exp[1:], t)
    c.free()


def test_captured_append_follows_the_lengths():
    c = Case([1, 1], [64, 64], page=8)
    cache, batch = c.cache(), c.batch()
    kb, vb = c.keep[0], c.keep[1]
    lens = c.keep[3]
    assert np.array_equal(lens.numpy(), c.kv_len)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, c.kv_heads, c.head)).astype(np.float32)
    d = c.put(x)
    cos, sin = tables(64, 32)
    cd, sd = c.put(cos), c.put(sin)

    def call():
        paged.append(cache, batch, None, d, d, cd, sd, None, heads=1, max_pos=64, half_rot=32,
                     ctx=c.ctx)

    call()
    c.ctx.synchronize()
    c.k_raw, c.v_raw = kb.numpy(), vb.numpy()
    c.ctx.graph_begin()
    call()
    g = c.ctx.graph_end()
    for step in ([1, 2], [9, 8], [33, 64]):
        c.kv_len = np.array(step, np.int32)
        lens.upload(c.kv_len)
        c.ctx.synchronize()
        c.ctx.graph_launch(g)
        c.ctx.synchronize()
        exp = want(c, (np.zeros((2, 1, c.head), np.float32), x, x, cos, sin))
        same((kb.numpy(), vb.numpy()), exp[1:], "f16")
        c.k_raw, c.v_raw = exp[1], exp[2]
    c.ctx.graph_destroy(g)
    c.free()
