"""Serving attention over a paged key/value cache, as cases that can be timed and compared.

Operators (``kind``):

* ``append``  rotary positions on the new rows' queries and keys, keys and values rounded to the
              cache's type and stored in their pages;
* ``attend``  attention of the new rows over their sequences' pages: single tokens and prompts,
              with a window, capped scores, a bias that falls with distance, a two-way prefix;
* ``shared``  the same where every sequence of the batch continues one long common prefix that
              the cache holds once.

Activations are binary32, as MatMulNBits gives and takes them; the cache is binary32, fp16 or
bf16.  A batch is ragged: sequence b's new rows are ``start[b] .. start[b + 1]``, they are the
last of its ``kv_len[b]`` keys, and key j lies in page ``pages[b, j // page]``, row ``j % page``
of a cache ``[num_pages, kv_heads, page, head]``.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # four sequences of a small model take one token each: launch latency
        dict(name="append_4", kind="append", batch=4, q=1, kv=700, ragged=True, heads=16,
             kv_heads=8, head=128, type="f16", page=16, rot=64, inter=False),
        # seven prompts of uneven length, half of each head rotated, pairs interleaved
        dict(name="append_prompts", kind="append", batch=7, q=1111, kv=1600, ragged=True, heads=32,
             kv_heads=8, head=64, type="bf16", page=64, rot=16, inter=True),
        # one long document at once
        dict(name="append_long", kind="append", batch=1, q=30001, kv=30001, ragged=False, heads=32,
             kv_heads=8, head=128, type="f16", page=64, rot=64, inter=False),
        # one user's next token after a short talk: launch latency
        dict(name="token_one", kind="attend", batch=1, q=1, kv=523, ragged=False, heads=16,
             kv_heads=8, head=128, type="f16", page=16, window=0, cap=0.0, bias=False, two=0.0),
        # the next tokens of a busy server's batch
        dict(name="token_batch", kind="attend", batch=64, q=1, kv=8192, ragged=True, heads=32,
             kv_heads=8, head=128, type="bf16", page=64, window=0, cap=0.0, bias=False, two=0.0),
        # the next tokens of two very long talks, scores capped
        dict(name="token_long", kind="attend", batch=2, q=1, kv=131071, ragged=True, heads=64,
             kv_heads=8, head=128, type="f16", page=128, window=0, cap=50.0, bias=False, two=0.0),
        # uneven prompts on a binary32 cache, a head of its own for each query, distance bias
        dict(name="prompt_uneven", kind="attend", batch=5, q=777, kv=1501, ragged=True, heads=12,
             kv_heads=12, head=96, type="f32", page=32, window=0, cap=0.0, bias=True, two=0.0),
        # a part of a prompt after what the cache holds, sliding window, two-way first part
        dict(name="prompt_window", kind="attend", batch=2, q=2048, kv=9000, ragged=True, heads=16,
             kv_heads=8, head=128, type="bf16", page=64, window=4096, cap=0.0, bias=False, two=0.1),
        # a long prompt at once
        dict(name="prompt_long", kind="attend", batch=1, q=8192, kv=8192, ragged=False, heads=32,
             kv_heads=8, head=128, type="f16", page=64, window=0, cap=0.0, bias=False, two=0.0),
        # a few answers to one question sampled side by side
        dict(name="shared_few", kind="shared", batch=6, q=1, prefix=509, kv=45, ragged=True,
             heads=16, kv_heads=8, head=128, type="f16", page=16, window=0, cap=0.0, bias=False,
             two=0.0),
        # a system prompt before every talk, heads of 64, scores capped
        dict(name="shared_talks", kind="shared", batch=33, q=1, prefix=4001, kv=700, ragged=True,
             heads=32, kv_heads=4, head=64, type="bf16", page=64, window=0, cap=30.0, bias=False,
             two=0.0),
        # many questions about one long document
        dict(name="shared_document", kind="shared", batch=128, q=1, prefix=32768, kv=512,
             ragged=True, heads=32, kv_heads=8, head=128, type="f16", page=64, window=0, cap=0.0,
             bias=False, two=0.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12])
    group = rng.choice([1, 2, 3, 4, 4, 8])
    c = dict(batch=1, q=1, kv=1, ragged=rng.random() < 0.8, heads=kv_heads * group,
             kv_heads=kv_heads, head=rng.choice([64, 96, 128, 128]),
             type=rng.choice(["f16", "f16", "bf16", "bf16", "f32"]),
             page=rng.choice([8, 16, 32, 64, 128]))
    f = rng.random()
    if f < 0.25:
        c["kind"] = "append"
        if rng.random() < 0.5:
            c.update(batch=_log(rng, 1, 256), kv=_log(rng, 1, 2048))
        else:
            c["batch"] = _log(rng, 1, 16)
            c["q"] = _log(rng, 2, 16384 // c["batch"])
            c["kv"] = c["q"] + rng.choice([0, _log(rng, 1, 2048)])
        c.update(rot=rng.choice([c["head"] // 2, c["head"] // 2, c["head"] // 4]),
                 inter=rng.random() < 0.3)
        return c
    c.update(window=0, cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.random() < 0.2,
             two=0.0 if rng.random() < 0.8 else round(rng.uniform(0.05, 0.6), 3))
    row = kv_heads * c["head"]  # values of one key
    if f < 0.5:
        c.update(kind="attend", batch=_log(rng, 1, 64))
        c["kv"] = _log(rng, 1, min(131072, (1 << 28) // (row * c["batch"])))
        if rng.random() < 0.2:
            c["q"] = min(c["kv"], rng.choice([2, 3, 5]))
    elif f < 0.75:
        c.update(kind="attend", batch=_log(rng, 1, 8))
        most = (1 << 30) // (c["batch"] * c["heads"])  # scores of one head and sequence
        c["q"] = _log(rng, 2, min(4096, math.isqrt(most)))
        c["kv"] = c["q"] + rng.choice([0, 0, _log(rng, 1, max(1, min(16384, most // c["q"]
                                                                      - c["q"])))])
    else:
        c.update(kind="shared", batch=_log(rng, 2, 128), prefix=_log(rng, 16, 32768),
                 kv=_log(rng, 1, 1024))
        if c["batch"] * c["heads"] * (c["prefix"] + c["kv"]) > 1 << 27:
            c["prefix"] = max(16, (1 << 27) // (c["batch"] * c["heads"]) - c["kv"])
    if rng.random() < 0.25:
        c["window"] = _log(rng, 16, 8192)
    return c


# ------------------------------------------------------------------ inputs
def _lengths(c):
    """New rows and keys of each sequence: a case's alone, so that its work is known."""
    q, kv = [], []
    for b in range(c["batch"]):
        f, g = (b * 0.6180339887498949) % 1.0, (b * 0.7548776662466927) % 1.0
        n = max(1, round(c["q"] * (1 - 0.75 * f))) if c["ragged"] else c["q"]
        past = c["kv"] - c["q"]
        q.append(n)
        kv.append(n + (round(past * (1 - 0.9 * g)) if c["ragged"] else past))
    return q, kv


def _two(c, kv):
    return int(c["two"] * (c.get("prefix", 0) + kv))


def prepare(case, seed):
    c, s = case, {"case": case}
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def whole(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    B, H, G, D, page = c["batch"], c["heads"], c["kv_heads"], c["head"], c["page"]
    ql, kl = _lengths(c)
    T, first, P = sum(ql), c.get("prefix", 0), -(-c.get("prefix", 0) // page)
    s["start"] = whole([0] + torch.tensor(ql).cumsum(0).tolist())
    s["kv_len"] = whole(kl)
    s["max_q"], s["max_kv"] = max(ql), max(kl)
    # pages in no order; each sequence has its own, the prefix's lie among them
    need = [-(-n // page) for n in kl]
    cols, total = max(need), sum(need) + P
    order = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.zeros(B, cols, dtype=torch.int32, device="cuda")
    have = torch.arange(cols, device="cuda") < whole(need)[:, None]
    table[have] = order[P:]
    s["pages"], s["prefix_pages"], s["prefix"] = table, order[:P].contiguous(), first
    t = TYPES[c["type"]]
    # some channels of the keys are far larger than the others, as in trained layers
    size = torch.ones(D, device="cuda")
    size[torch.randperm(D, generator=g, device="cuda")[:max(1, D // 32)]] = 4.0
    s["k"] = (normal(total, G, page, D) * size).to(t)
    s["v"] = normal(total, G, page, D).to(t)
    if c["kind"] == "append":
        # one row of the projections' output: queries, keys, values
        s["qkv"] = normal(T, (H + 2 * G) * D)
        r, far = c["rot"], s["max_kv"]
        angle = torch.outer(torch.arange(far, dtype=torch.float64, device="cuda"),
                            1e6 ** (-torch.arange(r, dtype=torch.float64, device="cuda") / r))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = normal(T, H * D) * 1.5
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H)
        s["two"] = whole([_two(c, n) for n in kl])
    s["out"] = torch.empty(T, H * D, device="cuda")
    if own:
        from onnx_runtime_dart_amd import paged
        s["lib"] = paged
        s["cache"] = paged.PagedCache(s["k"].data_ptr(), s["v"].data_ptr(), c["type"],
                                      num_pages=total, page_size=page, kv_heads=G, head_size=D)
        s["batch"] = paged.PagedBatch(s["start"].data_ptr(), s["kv_len"].data_ptr(),
                                      s["pages"].data_ptr(), batch=B, tokens=T, page_cols=cols,
                                      max_q=s["max_q"], max_kv=s["max_kv"])
        if c["kind"] != "append":
            s["scores"] = paged.Scores(softcap=c["cap"], window=c["window"],
                                       slopes=s["slopes"].data_ptr() if c["bias"] else None,
                                       two_way=s["two"].data_ptr() if c["two"] else None)
        # the library's stream does not wait for torch's, on which these were made
        torch.cuda.synchronize()
    return s


# ------------------------------------------------------------- plain forms
def _rows(s):
    """Sequence and place within it of each new row, and its position among the keys."""
    lens = (s["start"][1:] - s["start"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), lens)
    at = torch.arange(len(seq), device="cuda") - s["start"][seq]
    return seq, at, s["kv_len"][seq] - lens[seq] + at


def _append(s):
    c = s["case"]
    H, G, D, r = c["heads"], c["kv_heads"], c["head"], c["rot"]
    seq, _, pos = _rows(s)
    x = s["qkv"].view(-1, H + 2 * G, D)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    turned = x[:, :H + G].clone()
    if c["inter"]:
        a, b = x[:, :H + G, 0:2 * r:2], x[:, :H + G, 1:2 * r:2]
        turned[..., 0:2 * r:2], turned[..., 1:2 * r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[:, :H + G, :r], x[:, :H + G, r:2 * r]
        turned[..., :r], turned[..., r:2 * r] = a * cos - b * sin, b * cos + a * sin
    s["out"].copy_(turned[:, :H].reshape(-1, H * D))
    where = s["pages"][seq, pos // c["page"]].long(), pos % c["page"]
    s["k"][where[0], :, where[1]] = turned[:, H:].to(s["k"].dtype)
    s["v"][where[0], :, where[1]] = x[:, H + G:].to(s["v"].dtype)
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _keys(cache, pages, count):
    """[..., kv_heads, count, head] in 32 bits of the pages [..., n]."""
    x = cache[pages.long()].transpose(-4, -3)
    return x.reshape(*x.shape[:-3], -1, x.shape[-1])[..., :count, :].float()


def _attend(s):
    c = s["case"]
    B, H, G, D, P = c["batch"], c["heads"], c["kv_heads"], c["head"], s["prefix"]
    M, N, R = s["max_q"], s["max_kv"], c["heads"] // c["kv_heads"]
    seq, at, _ = _rows(s)
    q = torch.zeros(B, M, H * D, device="cuda")
    q[seq, at] = s["q"]
    q = q.view(B, M, G, R, D).permute(0, 2, 3, 1, 4).reshape(B, G, R * M, D)
    k, v = (_keys(s[x], s["pages"], N) for x in "kv")
    z = (q @ k.transpose(-1, -2)).view(B, G, R, M, N)
    if P:  # all sequences' rows over the prefix in one product
        pk, pv = (_keys(s[x], s["prefix_pages"], P) for x in "kv")
        flat = q.transpose(0, 1).reshape(G, B * R * M, D)
        zp = (flat @ pk.transpose(-1, -2)).view(G, B, R, M, P).transpose(0, 1)
        z = torch.cat((zp, z), -1)
    z = z * (1.0 / math.sqrt(D))
    if c["cap"]:
        z = c["cap"] * torch.tanh(z / c["cap"])
    lens = s["start"][1:] - s["start"][:-1]
    i = P + (s["kv_len"] - lens)[:, None, None] + torch.arange(M, device="cuda")[:, None]
    j = torch.arange(P + N, device="cuda")
    if c["bias"]:
        far = (i - j).abs().float()[:, None, None]
        z = z - s["slopes"].view(1, G, R, 1, 1) * far
    seen = j <= i
    if c["window"]:
        seen = seen & (j > i - c["window"])
    if c["two"]:
        seen = seen | (j < s["two"][:, None, None])
    seen = seen & (j < P + s["kv_len"][:, None, None])
    z = torch.where(seen[:, None, None], z, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top.isfinite(), top, 0.0))
    total = e.sum(-1).reshape(B, G, R * M, 1)
    o = e[..., P:].reshape(B, G, R * M, N) @ v
    if P:
        flat = e[..., :P].transpose(0, 1).reshape(G, B * R * M, P) @ pv
        o = o + flat.view(G, B, R * M, D).transpose(0, 1)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.view(B, G, R, M, D).permute(0, 3, 1, 2, 4).reshape(B, M, H * D)
    s["out"].copy_(o[seq, at])
    return s["out"]


def run(state):
    s = state
    c = s["case"]
    if not own:
        return _append(s) if c["kind"] == "append" else _attend(s)
    if c["kind"] == "append":
        D, ld = c["head"], s["qkv"].shape[1]
        at = s["qkv"].data_ptr()
        k = at + 4 * c["heads"] * D
        s["lib"].append(s["cache"], s["batch"], at, k, k + 4 * c["kv_heads"] * D,
                        s["cos"].data_ptr(), s["sin"].data_ptr(), s["out"].data_ptr(),
                        heads=c["heads"], max_pos=s["max_kv"], half_rot=c["rot"],
                        interleaved=c["inter"], ldq=ld, ldk=ld, ldv=ld)
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    if c["kind"] == "attend":
        s["lib"].attention(s["cache"], s["batch"], s["q"].data_ptr(), s["out"].data_ptr(),
                           heads=c["heads"], scores=s["scores"])
    else:
        s["lib"].attention_shared(s["cache"], s["batch"], s["prefix_pages"].data_ptr(),
                                  s["prefix"], s["q"].data_ptr(), s["out"].data_ptr(),
                                  heads=c["heads"], scores=s["scores"])
    return s["out"]


# ------------------------------------------------------- what a pass needs
def _span(c, n, kv, i):
    """Keys that row i of a sequence's n new ones sees: how many, and the first of the run that
    ends at its own place."""
    P = c.get("prefix", 0)
    at = P + kv - n + i
    lo = max(0, at - c["window"] + 1) if c["window"] else 0
    two = min(_two(c, kv), P + kv)
    return at + 1 - lo + max(0, min(two, lo)) + max(0, two - at - 1), lo


def work(case):
    c = case
    ql, kl = _lengths(c)
    T, H, G, D = sum(ql), c["heads"], c["kv_heads"], c["head"]
    size = 4 if c["type"] == "f32" else 2
    if c["kind"] == "append":
        places = len({kv - n + i for n, kv in zip(ql, kl) for i in range(n)})
        return {"bytes": T * D * (8 * H + G * (8 + 2 * size)) + places * c["rot"] * 8 + 12 * T,
                "flops": 6 * T * (H + G) * c["rot"]}
    pairs, keys, P, low = 0, 0, c.get("prefix", 0), c.get("prefix", 0)
    for n, kv in zip(ql, kl):
        seen = [_span(c, n, kv, i) for i in range(n)]
        pairs += sum(x[0] for x in seen)
        two, lo = min(_two(c, kv), P + kv), seen[0][1]
        # keys of its own that some row of the sequence sees, and what of the prefix
        keys += kv - max(0, lo - max(P, two)) if lo > P else kv
        low = min(low, lo if two <= 0 else max(0, lo - two))
    return {"bytes": (keys + P - low) * G * D * 2 * size + 8 * T * H * D,
            "flops": 4 * pairs * H * D}


# ------------------------------------------------------- in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    H, G, D, page, P = c["heads"], c["kv_heads"], c["head"], c["page"], s["prefix"]
    R = H // G
    ql, kl = _lengths(c)
    if c["kind"] == "append":
        k, v = s["k"].double(), s["v"].double()
        x = s["qkv"].double()
        q, r, row = x[:, :H * D].clone(), c["rot"], 0
        for b, (n, kv) in enumerate(zip(ql, kl)):
            pos = torch.arange(kv - n, kv, device="cuda")
            # a pair of values is a complex number, turned by the angle of its position
            turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]

            def turned(y):
                z = y.reshape(n, -1, D).clone()
                if c["inter"]:
                    pair = torch.view_as_complex(z[..., :2 * r].reshape(n, -1, r, 2).contiguous())
                    z[..., :2 * r] = torch.view_as_real(pair * turn).reshape(n, -1, 2 * r)
                else:
                    pair = torch.complex(z[..., :r], z[..., r:2 * r]) * turn
                    z[..., :r], z[..., r:2 * r] = pair.real, pair.imag
                return z

            y = x[row:row + n]
            q[row:row + n] = turned(y[:, :H * D]).reshape(n, H * D)
            p, o = s["pages"][b][pos // page].long(), pos % page
            k[p, :, o] = turned(y[:, H * D:(H + G) * D])
            v[p, :, o] = y[:, (H + G) * D:].reshape(n, G, D)
            row += n
        return {"q": q, "k": k, "v": v}
    out, row = torch.empty(sum(ql), H, D, dtype=torch.float64, device="cuda"), 0
    for b, (n, kv) in enumerate(zip(ql, kl)):
        in_page = torch.arange(page, device="cuda")
        at = torch.cat([(t.long()[:, None] * page + in_page).reshape(-1)[:count]
                        for t, count in ((s["prefix_pages"], P), (s["pages"][b], kv))])
        i = torch.arange(P + kv - n, P + kv, device="cuda")[:, None]
        j = torch.arange(P + kv, device="cuda")[None]
        keep = j <= i
        if c["window"]:
            keep &= i - j < c["window"]
        if c["two"]:
            keep |= j < _two(c, kv)
        for h in range(H):
            k, v = (s[x].transpose(0, 1)[h // R].reshape(-1, D)[at].double() for x in "kv")
            z = s["q"][row:row + n, h * D:(h + 1) * D].double() @ k.T / math.sqrt(D)
            if c["cap"]:
                z = torch.tanh(z / c["cap"]) * c["cap"]
            if c["bias"]:
                z -= s["slopes"][h].double() * (i - j).abs()
            out[row:row + n, h] = z.masked_fill_(~keep, -math.inf).softmax(-1) @ v
        row += n
    return out.view(-1, H * D)
