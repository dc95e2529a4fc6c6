"""Paged key/value cache: the batch's new rows stored in pages, and attention over them.

Python side of ``mmnb_paged_*`` (include/mmnb.h): descriptions of a cache, of a batch and of
the scores, and one function per entry point.  Everything is device memory and runs on the
context's stream without waiting.  A device buffer is given as a ``DeviceBuffer`` or as its
address (an integer), so that buffers of other libraries serve too.  The context's stream waits
for no other and no other for it: wait for another library's stream before a call reads what it
wrote, and ``ctx.synchronize()`` before that library reads a result.
"""
import ctypes

from . import _lib
from ._lib import check

TYPES = {"f32": _lib.DT_F32, "f16": _lib.DT_F16, "bf16": _lib.DT_BF16}


def _addr(x):
    """The address of a DeviceBuffer, an integer address, or None."""
    if x is None or isinstance(x, int):
        return x
    p = x.ptr
    return p.value if isinstance(p, ctypes.c_void_p) else p


class _Desc:
    """A C structure with the buffers that it points to kept alive."""

    def __init__(self, struct, *keep):
        self.struct = struct
        self.ref = ctypes.addressof(struct)
        self._keep = keep


class PagedCache(_Desc):
    """Keys and values in pages ``[num_pages, kv_heads, page_size, head_size]`` (or at
    ``strides = (page, head, row)``, in elements) of type "f32", "f16" or "bf16"."""

    def __init__(self, k, v, dtype, *, num_pages, page_size, kv_heads, head_size, strides=None):
        if dtype not in TYPES:
            raise NotImplementedError(f"paged cache: type must be one of {sorted(TYPES)}, "
                                      f"got {dtype}")
        s = tuple(int(x) for x in strides) if strides is not None else (0, 0, 0)
        if len(s) != 3:
            raise ValueError("paged cache: strides are (page, head, row)")
        super().__init__(_lib.PagedCache(_addr(k), _addr(v), TYPES[dtype], num_pages, page_size,
                                         kv_heads, head_size, *s), k, v)
        self.kv_width = kv_heads * head_size
        self.head_size = head_size


class PagedBatch(_Desc):
    """A ragged batch: ``start`` int32 [batch + 1], ``kv_len`` int32 [batch], ``pages`` int32
    [batch, page_cols]; ``max_q`` and ``max_kv`` bound the sequences' new rows and keys."""

    def __init__(self, start, kv_len, pages, *, batch, tokens, page_cols, max_q, max_kv):
        super().__init__(_lib.PagedBatch(batch, tokens, _addr(start), _addr(kv_len),
                                         _addr(pages), page_cols, max_q, max_kv),
                         start, kv_len, pages)


class Scores(_Desc):
    """How scores become softmax weights: scale (0: 1 / sqrt(head_size)), tanh cap, window,
    ``slopes`` fp32 [heads] of a bias that falls with distance, ``two_way`` int32 [batch] first
    keys that every row sees."""

    def __init__(self, scale=0.0, softcap=0.0, window=0, slopes=None, two_way=None):
        super().__init__(_lib.PagedScores(scale, softcap, window, _addr(slopes),
                                          _addr(two_way)), slopes, two_way)


def _ctx(ctx):
    return ctx if ctx is not None else _lib.default_context()


def append(cache, batch, q, k, v, cos, sin, q_out, *, heads, max_pos, half_rot,
           interleaved=False, first_pos=0, ldq=None, ldk=None, ldv=None, ldqo=None, ctx=None):
    """Stores the rows' keys and values (rotated keys) in their pages and writes the rotated
    queries to ``q_out``, which may be ``q``.  ``ld*``: floats from one row to the next (default:
    no gap, and ``ldq`` for queries turned in place)."""
    ctx = _ctx(ctx)
    qw, kw = heads * cache.head_size, cache.kv_width
    if ldqo is None and _addr(q_out) == _addr(q):
        ldqo = ldq
    check(ctx.lib.mmnb_paged_append_dev(
        ctx.handle, cache.ref, batch.ref, _addr(q), qw if ldq is None else ldq, heads, _addr(k),
        kw if ldk is None else ldk, _addr(v), kw if ldv is None else ldv, _addr(cos), _addr(sin),
        max_pos, half_rot, bool(interleaved), first_pos, _addr(q_out),
        qw if ldqo is None else ldqo))


def attention(cache, batch, q, out, *, heads, scores=None, ldq=None, ldo=None, ctx=None):
    """Attention of the batch's rows over their sequences' pages."""
    ctx = _ctx(ctx)
    w = heads * cache.head_size
    check(ctx.lib.mmnb_paged_attention_dev(
        ctx.handle, cache.ref, batch.ref, None if scores is None else scores.ref, _addr(q),
        w if ldq is None else ldq, heads, _addr(out), w if ldo is None else ldo))


def attention_shared(cache, batch, prefix_pages, prefix_len, q, out, *, heads, scores=None,
                     ldq=None, ldo=None, ctx=None):
    """The same for sequences that all continue the ``prefix_len`` keys in ``prefix_pages``."""
    ctx = _ctx(ctx)
    w = heads * cache.head_size
    check(ctx.lib.mmnb_paged_attention_shared_dev(
        ctx.handle, cache.ref, batch.ref, _addr(prefix_pages), prefix_len,
        None if scores is None else scores.ref, _addr(q), w if ldq is None else ldq, heads,
        _addr(out), w if ldo is None else ldo))
