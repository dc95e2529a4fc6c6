"""Paged cache operators in 64 bits, from their definition (include/mmnb.h).

TEST INFRASTRUCTURE ONLY, like the other modules here.  Caches are float64 arrays
``[num_pages, kv_heads, page, head]`` holding what the device's cache holds.
"""
import numpy as np


def rows(start, kv_len):
    """(sequence, row, key of its own) of every new row."""
    for b in range(len(kv_len)):
        n = int(start[b + 1]) - int(start[b])
        for i in range(n):
            yield b, int(start[b]) + i, int(kv_len[b]) - n + i


def rotate(x, cos, sin, interleaved):
    """x [heads, head] turned by one position's cos/sin [half], in double, as binary32."""
    x = np.asarray(x, np.float64)
    y, r = x.copy(), len(cos)
    c, s = np.asarray(cos, np.float64), np.asarray(sin, np.float64)
    lo, hi = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved else (slice(0, r),
                                                                          slice(r, 2 * r))
    y[:, lo] = x[:, lo] * c - x[:, hi] * s
    y[:, hi] = x[:, hi] * c + x[:, lo] * s
    return y.astype(np.float32)


def keys_of(cache, pages, count, g):
    """[count, head] of key/value head g."""
    page = cache.shape[2]
    j = np.arange(count)
    return cache[np.asarray(pages)[j // page], g, j % page]


def attend(q, k, v, start, kv_len, pages, *, prefix_pages=(), prefix=0, scale=0.0, cap=0.0,
           window=0, slopes=None, two=None, split_bits=24):
    """(out, tol): the operator in 64 bits for q [tokens, heads, head], and how far a result
    in 32-bit arithmetic may be off.

    tol, from the roundings (each at most u = 2^-24 relative; independent, so that sums of n
    of them grow as sqrt(n); four standard deviations):
      a product of `head` terms: 4 u sqrt(head + 8) |(q_d k_d)_d|, and the split of q to
      `split_bits` bits another 4 2^-split_bits |(q_d k_d)_d|; scaling, cap, bias and the
      exponent's argument 8 u max|z|; a capped score besides 8 u cap (tanh's own rounding);
      a weight: that, 4 u for the exponential and 2^-split_bits for its split;
      an output: sum_j p_j |v_j| times twice a weight's error (numerator and denominator),
      and 4 u sqrt(keys) for the sums."""
    T, H, D = q.shape
    G = k.shape[1]
    u, sb = 2.0 ** -24, 2.0 ** -split_bits
    scale = scale if scale > 0 else 1.0 / np.sqrt(D)
    out, tol = np.zeros((T, H, D)), np.zeros((T, H, D))
    q = np.asarray(q, np.float64)
    for b, t, own in rows(start, kv_len):
        p, total = prefix + own, prefix + int(kv_len[b])
        j = np.arange(total)
        seen = (j <= p) & ((j > p - window) if window else True)
        if two is not None:
            seen |= j < int(two[b])
        j = j[seen]
        if not len(j):
            continue
        for g in range(G):
            kk, vv = (np.concatenate([keys_of(c, prefix_pages, prefix, g),
                                      keys_of(c, pages[b], int(kv_len[b]), g)])[j]
                      for c in (k, v))
            for h in range(g * (H // G), (g + 1) * (H // G)):
                with np.errstate(all="ignore"):
                    prod = q[t, h] * kk
                    z = prod.sum(-1) * scale
                    live = np.isfinite(z)  # the others weigh nothing, or the row is NaN
                    size = np.sqrt((prod[live] ** 2).sum(-1)).max(initial=0.0) * scale
                    if cap:
                        z = cap * np.tanh(z / cap)
                    if slopes is not None:
                        z = z - float(slopes[h]) * np.abs(p - j)
                    top = z.max()
                    e = np.exp(z - (top if top != -np.inf else 0.0))
                    w = e / e.sum() if e.sum() != 0 else 0 * e
                    out[t, h] = w @ vv if np.isfinite(vv).all() else (w[:, None] * vv).sum(0)
                    dz = 4 * (u * np.sqrt(D + 8) + sb) * size
                    dz += 8 * u * (np.abs(z[live]).max(initial=0.0) + cap)
                    dw = dz + 4 * u + sb
                    tol[t, h] = (2 * dw + 4 * u * np.sqrt(len(j))) * \
                        (w[live] @ np.abs(vv[live])) + 1e-37
    return out, tol
