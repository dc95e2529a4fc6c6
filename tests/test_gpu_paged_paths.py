"""Paged attention where the launches take each of their forms: batches beyond a wave's lanes,
sequences cut or whole, tiles of 64 and 128 rows, parts of the keys, prefixes among the sequences
and apart.  The reference is the definition in 64 bits, computed densely on the device."""
import math

import numpy as np
import pytest
import torch

from tests.paged_cases import SPLIT_BITS, Case, close

pytestmark = pytest.mark.gpu

TYPES = ["f16", "bf16", "f32"]


def dense(c):
    """(out, tol) as oracle.paged.attend has them (its tolerance's derivation is there), for
    caches without infinities and NaN."""
    dev, H, G, D = "cuda", c.heads, c.kv_heads, c.head
    u, sb = 2.0 ** -24, 2.0 ** -SPLIT_BITS[c.t]
    scale = c.scale if c.scale > 0 else 1.0 / math.sqrt(D)
    k, v = (torch.from_numpy(x).to(dev) for x in (c.k, c.v))
    q = torch.from_numpy(c.q).to(dev).double()
    out, tol = torch.zeros_like(q), torch.zeros_like(q)

    def rows(x, pages, n, g):
        j = torch.arange(n, device=dev)
        return x[torch.from_numpy(np.asarray(pages)).to(dev).long()[j // c.page], g, j % c.page]

    for b in range(len(c.kv_len)):
        r0, r1, n = int(c.start[b]), int(c.start[b + 1]), int(c.kv_len[b])
        if r0 == r1:
            continue
        p = c.prefix + torch.arange(n - (r1 - r0), n, device=dev)[:, None]
        j = torch.arange(c.prefix + n, device=dev)[None]
        seen = j <= p
        if c.window:
            seen &= j > p - c.window
        if c.two is not None:
            seen |= j < int(c.two[b])
        for g in range(G):
            kk, vv = (torch.cat([rows(x, c.prefix_pages, c.prefix, g),
                                 rows(x, c.pages[b], n, g)]) for x in (k, v))
            hs = slice(g * (H // G), (g + 1) * (H // G))
            y = q[r0:r1, hs].transpose(0, 1)  # [heads, rows, head]
            z = y @ kk.T * scale
            size = ((y * y) @ (kk * kk).T).clamp_min(0).sqrt() * scale
            if c.cap:
                z = c.cap * torch.tanh(z / c.cap)
            if c.slopes is not None:
                slopes = torch.from_numpy(c.slopes[hs]).to(dev).double()
                z = z - slopes[:, None, None] * (p - j).abs()
            big = torch.where(seen, z.abs(), 0.0).amax(-1, keepdim=True)
            size = torch.where(seen, size, 0.0).amax(-1, keepdim=True)
            w = z.masked_fill(~seen, -math.inf).softmax(-1)
            dz = 4 * (u * math.sqrt(D + 8) + sb) * size + 8 * u * (big + c.cap)
            count = seen.sum(-1, keepdim=True).double()
            out[r0:r1, hs] = (w @ vv).transpose(0, 1)
            tol[r0:r1, hs] = ((2 * (dz + 4 * u + sb) + 4 * u * count.sqrt()) *
                              (w @ vv.abs()) + 1e-37).transpose(0, 1)
    return out.cpu().numpy(), tol.cpu().numpy()


def check(c):
    y = c.run()
    want, tol = dense(c)
    c.free()
    close(y, want, tol)


MODS = [{}, dict(cap=7.0, bias=True), dict(window=150, bias=True)]


@pytest.mark.parametrize("t", TYPES)
def test_the_dense_reference_is_the_definition(t):
    c = Case([5, 3], [40, 3], t=t, prefix=19, cap=6.0, window=20, bias=True, two=[3, 30])
    want, tol = c.want()
    got, gtol = dense(c)
    assert np.allclose(got, want, rtol=0, atol=1e-12) and np.allclose(gtol, tol, rtol=1e-9)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mod", MODS)
@pytest.mark.parametrize("kv", [1, 33, 161])
def test_tokens_of_many_sequences(t, mod, kv):
    """Seventy sequences, whole in a wave or cut."""
    kvs = [max(1, kv - (i * 7) % (kv + 3)) for i in range(70)]
    check(Case([1] * 70, kvs, t=t, heads=6, kv_heads=3, head=128, page=32, max_kv=kv, **mod))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kv", [500, 520])
def test_tokens_of_more_pairs_than_half_the_waves(t, kv):
    kvs = [kv - 13 * i for i in range(33)]
    check(Case([1] * 33, kvs, t=t, heads=16, kv_heads=16, head=128, page=64))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mod", MODS)
@pytest.mark.parametrize("new", [[600], [300, 1, 290], [9] * 66])
def test_prompts_in_tiles_of_64_rows(t, mod, new):
    check(Case(new, [n + 37 for n in new], t=t, heads=32, kv_heads=32, head=64, page=16, **mod))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("head", [64, 96, 128])
@pytest.mark.parametrize("new,kv", [([801], [801]), ([500, 0, 400], [900, 50, 400]),
                                    ([1100, 700], [1100, 1000])])
def test_prompts_in_tiles_of_128_rows(t, head, new, kv):
    check(Case(new, kv, t=t, heads=64, kv_heads=32, head=head, page=64))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mod", MODS + [dict(window=300, two=[700, 3])])
def test_windows_over_prompts_in_tiles_of_128_rows(t, mod):
    check(Case([700, 230], [1300, 800], t=t, heads=64, kv_heads=32, head=128, page=32, **mod))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mod", MODS)
@pytest.mark.parametrize("new,kv", [([64], [1100]), ([200, 33], [2300, 1700]), ([40], [129])])
def test_prompts_on_eight_waves_a_tile(t, mod, new, kv):
    check(Case(new, kv, t=t, heads=4, kv_heads=2, head=128, page=16, **mod))
    check(Case(new, kv, t=t, heads=4, kv_heads=2, head=72, page=16, **mod))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mod", MODS)
@pytest.mark.parametrize("step", [2, 5])
def test_prefix_in_tiles_of_64_rows(t, mod, step):
    """128 rows of a head over 3000 keys of 16 heads: more than the waves take by themselves.
    The sequences' own keys in the same launch, or too many for it."""
    check(Case([1] * 32, [1 + step * i for i in range(32)], t=t, heads=64, kv_heads=16, head=128,
               page=64, prefix=3000, **mod))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("head,mod", [(64, MODS[0]), (128, MODS[1]), (64, MODS[2])])
def test_prefix_in_tiles_of_128_rows(t, head, mod):
    check(Case([1] * 50, [1 + 3 * i for i in range(50)], t=t, heads=64, kv_heads=16, head=head,
               page=64, prefix=9001, **mod))


@pytest.mark.parametrize("t", TYPES)
def test_prefix_in_tiles_of_128_rows_before_several_rows_of_a_sequence(t):
    check(Case([0, 4, 1, 3] * 13, [9, 4, 700, 100] * 13, t=t, heads=32, kv_heads=16, head=96,
               page=16, prefix=9001))
    check(Case([0, 4, 1, 3] * 13, [9, 4, 400, 100] * 13, t=t, heads=64, kv_heads=16, head=96,
               page=16, prefix=9001, bias=True))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mod", MODS)
@pytest.mark.parametrize("batch,group,prefix", [(3, 5, 700), (90, 1, 333), (33, 8, 1000)])
def test_prefix_among_the_sequences(t, mod, batch, group, prefix):
    check(Case([1] * batch, [1 + i % 70 for i in range(batch)], t=t, heads=2 * group, kv_heads=2,
               head=96, page=16, prefix=prefix, **mod))


@pytest.mark.parametrize("t", TYPES)
def test_prefix_before_prompts(t):
    check(Case([50, 3], [90, 3], t=t, heads=6, kv_heads=2, head=128, page=16, prefix=700))
    check(Case([300] * 2, [300, 400], t=t, heads=32, kv_heads=32, head=64, page=64, prefix=130,
               window=200, two=[5, 500]))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("prefix,batch,heads,kv_heads", [(300, 8, 4, 2), (3000, 32, 64, 16)])
def test_a_bad_page_of_the_prefix_or_of_a_sequence(t, prefix, batch, heads, kv_heads):
    for what in ("prefix", "own"):
        c = Case([1] * batch, [40] * batch, t=t, heads=heads, kv_heads=kv_heads, head=64,
                 page=16, prefix=prefix)
        pages = c.prefix_pages if what == "prefix" else c.pages[3]
        good = int(pages[1])
        pages[1] = -7
        y = c.run()
        pages[1] = good
        want, tol = dense(c)
        c.free()
        if what == "prefix":
            assert np.isnan(y).all()
        else:
            assert np.isnan(y[3]).all()
            rest = np.arange(batch) != 3
            close(y[rest], want[rest], tol[rest])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("prefix,batch,heads,kv_heads", [(300, 8, 4, 2), (3000, 32, 64, 16)])
def test_nan_in_the_prefix_reaches_the_rows_that_see_it(t, prefix, batch, heads, kv_heads):
    c = Case([1] * batch, [1 + i for i in range(batch)], t=t, heads=heads, kv_heads=kv_heads,
             head=64, page=16, prefix=prefix, window=40)
    page, at = c.prefix_pages[(prefix - 35) // 16], (prefix - 35) % 16
    bits = np.float32("nan") if t == "f32" else {"f16": 0x7e00, "bf16": 0x7fc0}[t]
    c.v_raw[page, 0, at, 9] = bits
    y = c.run()
    want, tol = dense(c)
    c.free()
    sees = (prefix + np.arange(batch)) - (prefix - 35) < 40
    group = heads // kv_heads
    assert sees.any() and not sees.all()
    assert np.isnan(y[sees][:, :group, 9]).all()
    y[:, :group, 9] = want[:, :group, 9]
    close(y, want, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new,kv", [([5] * 70, [60] * 70), ([1] * 70, [60] * 70),
                                    ([300, 200, 5], [300, 900, 5])])
def test_lengths_that_break_the_promises_in_any_form(t, new, kv):
    heads, kv_heads = (64, 32) if len(new) == 3 else (8, 2)
    c = Case(new, kv, t=t, heads=heads, kv_heads=kv_heads, head=64)
    want, tol = dense(c)
    c.kv_len[1] = 1 << 30
    y = c.run()
    c.free()
    a, b = c.start[1], c.start[2]
    assert np.isnan(y[a:b]).all()
    keep = np.r_[0:a, b:c.tokens]
    close(y[keep], want[keep], tol[keep])


@pytest.mark.parametrize("kw", [
    dict(new=[70], kv=[3000], heads=4, kv_heads=1, head=128),
    dict(new=[1] * 32, kv=[9] * 32, heads=64, kv_heads=16, head=128, prefix=3000),
    dict(new=[1] * 40, kv=[30] * 40, heads=8, kv_heads=2, head=64, prefix=100),
    dict(new=[300], kv=[900], heads=64, kv_heads=32, head=64)])
def test_captured_calls_of_every_form(kw):
    c = Case(**kw, t="bf16", page=64)
    call = c.device()
    call()
    c.ctx.synchronize()
    first = c.read().copy()
    c.ctx.graph_begin()
    call()
    g = c.ctx.graph_end()
    for _ in range(3):
        c.out.upload(np.full(c.out.shape, 7.0, np.float32))
        c.ctx.synchronize()
        c.ctx.graph_launch(g)
        c.ctx.synchronize()
        assert np.array_equal(c.read(), first)
        call()  # eager work between the replays
        c.ctx.synchronize()
        assert np.array_equal(c.read(), first)
    want, tol = dense(c)
    c.ctx.graph_destroy(g)
    c.free()
    close(first, want, tol)


def test_rows_in_no_sequence_are_left_alone():
    for heads, kv_heads, n in ((4, 2, 1), (4, 2, 40)):
        c = Case([n, n, n], [n + 50] * 3, heads=heads, kv_heads=kv_heads)
        want, tol = dense(c)
        c.start[:] = c.start + 2          # the call has two rows more before and after
        c.tokens += 4
        c.q = np.concatenate([c.q[:2], c.q, c.q[:2]])
        y = c.run()
        c.free()
        assert (y[:2] == 7.0).all() and (y[-2:] == 7.0).all()
        close(y[2:-2], want, tol)
