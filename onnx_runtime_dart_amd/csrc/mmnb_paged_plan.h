// What a call on a paged key/value cache is checked for, and where its rows and keys lie.
// Plain C++ that the kernels include too, so that the checks and the arithmetic on device
// data (lengths and page numbers that the host never sees) can be tested on the CPU.
#pragma once

#include <cfloat>
#include <cmath>
#include <cstdint>

#include "../../include/mmnb.h"

#ifdef __HIP__
#define MMNB_HD __host__ __device__ __forceinline__
#else
#define MMNB_HD inline
#endif

namespace mmnb {

constexpr int64_t kPagedMaxHead = 128;       // head size
constexpr int64_t kPagedMaxPage = 65536;     // rows of a page
constexpr int64_t kPagedMaxLen = 1 << 30;    // keys of a sequence, positions, rows of a call

struct PagedCheck {
  int code = MMNB_OK;
  const char *what = "";
};

inline PagedCheck paged_arg(const char *what) { return {MMNB_ERR_ARG, what}; }
inline PagedCheck paged_unsupported(const char *what) { return {MMNB_ERR_UNSUPPORTED, what}; }

// Where a cache's values lie, in elements.
struct PagedStrides {
  int64_t page = 0, head = 0, row = 0;
};
inline PagedStrides paged_strides(const mmnb_paged_cache &c) {
  if (c.stride_page || c.stride_head || c.stride_row)
    return {c.stride_page, c.stride_head, c.stride_row};
  return {c.kv_heads * c.page_size * c.head_size, c.page_size * c.head_size, c.head_size};
}

inline PagedCheck paged_check_cache(const mmnb_paged_cache *c) {
  if (!c) return paged_arg("null cache");
  if (c->type != MMNB_DT_F32 && c->type != MMNB_DT_F16 && c->type != MMNB_DT_BF16)
    return paged_unsupported("cache type must be float32, float16 or bfloat16");
  if (c->num_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->head_size <= 0)
    return paged_arg("cache shape must be positive");
  if (c->num_pages > INT32_MAX || c->kv_heads > 65535)
    return paged_unsupported("too many pages or heads");
  if ((c->page_size & (c->page_size - 1)) || c->page_size > kPagedMaxPage)
    return paged_unsupported("page_size must be a power of two up to 65536");
  if (c->head_size % 8 || c->head_size > kPagedMaxHead)
    return paged_unsupported("head_size must be a multiple of 8 up to 128");
  const PagedStrides s = paged_strides(*c);
  if (s.page <= 0 || s.head <= 0 || s.row < c->head_size)
    return paged_arg("cache strides must be positive and rows may not overlap");
  if (s.page % 8 || s.head % 8 || s.row % 8)
    return paged_unsupported("cache strides must be multiples of 8 elements");
  if (s.page > (int64_t(1) << 40) || s.head > (int64_t(1) << 40) || s.row > (int64_t(1) << 40))
    return paged_unsupported("cache strides above 2^40");
  if (!c->k || !c->v) return paged_arg("null cache buffer");
  if (((uintptr_t)c->k | (uintptr_t)c->v) % 16)
    return paged_arg("cache buffers must be aligned to 16 bytes");
  return {};
}

inline PagedCheck paged_check_batch(const mmnb_paged_cache &c, const mmnb_paged_batch *b) {
  if (!b) return paged_arg("null batch");
  if (b->batch < 0 || b->tokens < 0 || b->page_cols < 0 || b->max_q < 0 || b->max_kv < 0)
    return paged_arg("negative size in the batch");
  if (b->batch > 65535) return paged_unsupported("more than 65535 sequences");
  if (b->tokens > kPagedMaxLen || b->max_kv > kPagedMaxLen || b->page_cols > INT32_MAX)
    return paged_unsupported("more than 2^30 rows or keys");
  if (b->max_q > b->max_kv) return paged_arg("max_q above max_kv: new rows are keys too");
  if (b->max_kv > b->page_cols * c.page_size)
    return paged_arg("max_kv above what page_cols pages hold");
  if (b->batch && b->tokens) {
    if (!b->d_start || !b->d_kv_len) return paged_arg("null batch buffer");
    if (!b->d_pages && b->max_kv) return paged_arg("null page table");
  }
  return {};
}

// Rows of `heads` heads, ld apart.
inline PagedCheck paged_check_rows(const mmnb_paged_cache &c, int64_t heads, int64_t ld) {
  if (heads <= 0 || heads > 65535) return paged_arg("bad number of heads");
  if (ld < heads * c.head_size) return paged_arg("row stride below the heads' size");
  if (ld > (int64_t(1) << 40)) return paged_unsupported("row stride above 2^40");
  return {};
}

inline PagedCheck paged_check_rope(const mmnb_paged_cache &c, const mmnb_paged_batch &b,
                                   const float *d_cos, const float *d_sin, int64_t max_pos,
                                   int64_t half_rot, int64_t first_pos) {
  if (half_rot < 0 || 2 * half_rot > c.head_size) return paged_arg("rotary dim above head_size");
  if (half_rot && (!d_cos || !d_sin || max_pos <= 0)) return paged_arg("rotary tables");
  if (first_pos < 0) return paged_arg("negative first position");
  if (first_pos > kPagedMaxLen || first_pos + b.max_kv > kPagedMaxLen)
    return paged_unsupported("positions above 2^30");
  return {};
}

// Queries turned in place: an item is read whole before it is written, so a row may take its own
// place, but not (a part of) another's.  Rows of `width` floats, ld apart, of the inputs and of
// the outputs must be the same ones or have nothing in common.
inline PagedCheck paged_check_in_place(const float *in, int64_t ldi, const float *out, int64_t ldo,
                                       int64_t width, int64_t rows) {
  const __int128 a = (intptr_t)in, b = (intptr_t)out, size = 4;  // (strides go up to 2^40)
  if (rows < 1 || (a == b && (ldi == ldo || rows == 1))) return {};
  const __int128 last = rows - 1;
  if (a + (last * ldi + width) * size <= b || b + (last * ldo + width) * size <= a) return {};
  if (ldi == ldo) {  // columns of the same rows
    const __int128 row = ldi * size, off = (a > b ? a - b : b - a) % row;
    if (off >= width * size && off + width * size <= row) return {};
  }
  return paged_arg("q_out overlaps q: it must be q itself, with the same row stride, or apart");
}

inline PagedCheck paged_check_heads(const mmnb_paged_cache &c, int64_t heads) {
  if (heads % c.kv_heads) return paged_arg("num_heads is no multiple of kv_heads");
  return {};
}

// Rows of all heads are counted in 32 bits (the last 128 of them are a tile's).
inline PagedCheck paged_check_size(const mmnb_paged_batch &b, int64_t heads) {
  if (b.tokens * heads > INT32_MAX - 128) return paged_unsupported("more than 2^31 rows of heads");
  return {};
}

MMNB_HD bool paged_finite(float x) { return x - x == 0.0f; }

inline PagedCheck paged_check_scores(const mmnb_paged_scores *s) {
  if (!s) return {};
  if (!paged_finite(s->scale) || !paged_finite(s->softcap) || s->softcap < 0)
    return paged_arg("scale and softcap must be finite, softcap not negative");
  if (s->window < 0) return paged_arg("negative window");
  return {};
}

// A score in base 2 of a product q.k: mul tanh(in_mul q.k) with a cap, else mul q.k.
struct PagedFactors {
  bool capped;
  float mul, in_mul;
};
inline PagedFactors paged_factors(const mmnb_paged_scores *s, int64_t head_size) {
  const double scale = s && s->scale > 0.0f ? (double)s->scale
                                            : (double)(float)(1.0 / std::sqrt((double)head_size));
  PagedFactors f;
  // A cap past 2^100 changes no score below 2^88, and scale / cap would leave binary32's normal
  // numbers, as the factor itself its range: none.
  f.capped = s && s->softcap > 0.0f && s->softcap <= 0x1p100f;
  const double mul = (f.capped ? (double)s->softcap : scale) * 1.4426950408889634;
  const double in_mul = f.capped ? scale / (double)s->softcap : 0.0;
  f.mul = (float)(mul < FLT_MAX ? mul : FLT_MAX);  // finite, so that a product of 0 is 0
  f.in_mul = (float)(in_mul < FLT_MAX ? in_mul : FLT_MAX);
  return f;
}

inline PagedCheck paged_check_prefix(const mmnb_paged_batch &b, const int32_t *d_pages,
                                     int64_t len) {
  if (len < 0) return paged_arg("negative prefix length");
  if (len > kPagedMaxLen || len + b.max_kv > kPagedMaxLen)
    return paged_unsupported("more than 2^30 rows or keys");
  if (len && !d_pages) return paged_arg("null prefix page table");
  return {};
}

// One sequence as the device arrays describe it: n rows from row0 on, the last of len keys.
// Values that no batch may hold (rows outside the call's, a length below the rows' number or
// above the promised max_kv, more rows than max_q) leave `bad` set, with row0 and n still
// inside the call's rows.
struct PagedSeq {
  int row0, n, len;
  bool bad;
};
MMNB_HD PagedSeq paged_seq(int start, int end, int len, int64_t tokens, int64_t max_q,
                           int64_t max_kv) {
  PagedSeq s;
  s.bad = start < 0 || end < start || end > tokens || len < 0 || len > max_kv;
  s.row0 = start < 0 ? 0 : start > tokens ? (int)tokens : start;
  const int e = end < s.row0 ? s.row0 : end > tokens ? (int)tokens : end;
  s.n = e - s.row0;
  s.bad = s.bad || s.n > len || s.n > max_q;
  s.len = s.bad ? 0 : len;
  return s;
}

// Whether row t of the call is one of the sequence's.  Row t is looked for among starts that the
// batch promises to rise; where they do not, what a count or a search of them finds may hold
// other rows, and t - row0 would be no place in it.
MMNB_HD bool paged_in(const PagedSeq &s, int t) { return t >= s.row0 && t < s.row0 + s.n; }
MMNB_HD bool paged_holds(const int32_t *start, int b, int t) {
  return start[b] <= t && t < start[b + 1];
}

// A page number as the device array holds it, made safe to read from.
MMNB_HD int paged_page(int page, int num_pages, bool *bad) {
  const bool out = page < 0 || page >= num_pages;
  *bad = *bad || out;
  return out ? 0 : page;
}

// ---- how attention is cut into pieces of work
constexpr int kPagedTokenTile = 32;   // keys of a tile where a wave has rows of its own
// Floats of a wave's row in the merge's LDS: sums, m and l; whole vectors of four, as the sums
// are stored, so that every row begins at a multiple of 16 bytes.
constexpr int kPagedMergeRow = kPagedMaxHead + 4;
constexpr int kPagedTokenRows = 32;   // rows of a sequence and kv head that a wave takes

// `total` tiles of all sequences and heads in one line, dealt to `most` workers in equal runs:
// worker w has [w * each, (w + 1) * each).
MMNB_HD int paged_each(int total, int most) {
  return (int)(((uint32_t)total + (uint32_t)most - 1) / (uint32_t)most);
}
// Keys [lo, lo + n * tile) of its own that a sequence's rows see, lo a multiple of `tile`, with
// `two` the keys that all see, counted past the shared prefix.  A sequence that breaks the
// promises has one tile, in which its rows are set.
struct PagedRange {
  int lo, n;
};
MMNB_HD PagedRange paged_range(const PagedSeq &s, int window, int two, int tile) {
  if (s.n == 0) return {0, 0};
  if (s.bad) return {0, 1};
  int lo = 0;
  if (window > 0 && two <= 0) {
    lo = s.len - s.n - window + 1;  // of the first row
    lo = lo < 0 ? 0 : lo / tile * tile;
  }
  return {lo, (s.len - lo + tile - 1) / tile};
}

// The keys that a workgroup's rows see, in tiles: na tiles of the shared prefix from key loa on,
// then nb of the sequence's own from lob on, those below `own`.  The rows are `count` of the
// sequence's rows and a head's group in one line, from `first` on; `two` is counted from the
// prefix's begin.
struct PagedKeys {
  int loa, na, lob, nb, own;
};
MMNB_HD PagedKeys paged_keys(const PagedSeq &s, int prefix, int group, int window, int two,
                             int first, int count, int tile) {
  const int p = prefix + s.len - s.n;                // position of the sequence's first row
  const int p0 = p + first / group;
  int p1 = p + (first + count - 1) / group;
  if (p1 > prefix + s.len - 1) p1 = prefix + s.len - 1;
  const int from = window > 0 && two <= 0 && p0 >= window ? p0 - window + 1 : 0;
  int end = p1 + 1 > two ? p1 + 1 : two;
  if (end > prefix + s.len) end = prefix + s.len;
  PagedKeys k;
  k.own = end > prefix ? end - prefix : 0;
  k.loa = (from < prefix ? from : prefix) / tile * tile;
  k.lob = (from > prefix ? from - prefix : 0) / tile * tile;
  k.na = (prefix - k.loa + tile - 1) / tile;
  k.nb = k.own > k.lob ? (k.own - k.lob + tile - 1) / tile : 0;
  return k;
}

// Workgroups of `rows` rows that a sequence's take (one sets the rows of a sequence that breaks
// the promises).
MMNB_HD int paged_tiles_of(const PagedSeq &s, int group, int rows) {
  return s.n == 0 ? 0 : s.bad ? 1 : (s.n * group + rows - 1) / rows;
}
// The most that a call's sequences may take.
inline int64_t paged_row_tiles(int64_t batch, int64_t tokens, int64_t max_q, int64_t group,
                               int64_t rows) {
  int64_t each = (max_q * group + rows - 1) / rows;
  if (each < 1) each = 1;
  const int64_t a = batch * each, b = tokens * group / rows + batch;
  return a < b ? a : b;
}
// Keys of a prefix that no row sees lie below this multiple of 64, one that leaves some: a window
// reaches back from a place behind the prefix, unless `two` gives every row the first keys.
MMNB_HD int paged_prefix_seen(int prefix, int window, bool two) {
  if (window == 0 || two || window >= prefix) return 0;
  const int lo = prefix - window + 1;
  return (lo < prefix ? lo : prefix - 1) / 64 * 64;
}

// Page numbers outside the cache, of those looked at: the position of the last such page's first
// key (-1: none).  Rows, the first of them at position p, miss a key if their windows reach a
// position of that page or `two` keys are seen by all: pages before every window may have been
// given back.
MMNB_HD int paged_lose(int last, bool out, int page, int shift, int off) {
  const int at = out ? (page << shift) + off : -1;
  return at > last ? at : last;
}
MMNB_HD bool paged_missed(int last, int shift, int p, int window, int two) {
  const int from = window > 0 && two <= 0 && p >= window ? p - window + 1 : 0;
  return last >= 0 && last > from - (1 << shift);
}
// Keys [lo, hi) of all that hold those the row at position p sees.
struct PagedSpan {
  int lo, hi;
};
MMNB_HD PagedSpan paged_row_span(int p, int window, int two, int keys) {
  const int hi = p + 1 > two ? p + 1 : two;
  return {window > 0 && two <= 0 && p >= window ? p - window + 1 : 0, hi < keys ? hi : keys};
}

// How many of a sequence's tiles of `rows` rows end (their last row's place, counted from 1)
// behind key x; a sequence that breaks the promises is one that ends at the first key.
MMNB_HD int paged_tiles_behind(const PagedSeq &s, int group, int rows, int x) {
  const int all = paged_tiles_of(s, group, rows);
  if (s.bad) return x < 1 ? all : 0;
  const int y = x - (s.len - s.n);
  return y <= 0 ? all : y >= s.n ? 0 : all - y * group / rows;
}

// Parts that the keys of each of `blocks` workgroups are cut into, of `tiles` tiles and with at
// least `least` of them in a part, for `most` workgroups at a time.
inline int64_t paged_splits(int64_t blocks, int64_t tiles, int64_t least, int64_t most) {
  int64_t s = most / blocks;
  if (s > tiles / least) s = tiles / least;
  if (s < 1) s = 1;
  const int64_t each = (tiles + s - 1) / s;
  return each > 0 ? (tiles + each - 1) / each : 1;
}

// Parts for a prompt's keys, `tiles` tiles that a workgroup takes `groups` at a time, where
// `most` workgroups run at a time and the pieces of a part are `bytes`: the number with the
// least time, a round of tiles taking 1.6 us, the merge 6 and the pieces' way through memory and
// back 1 us for each MB.
inline int64_t paged_prompt_parts(int64_t blocks, int64_t tiles, int64_t groups, int64_t bytes,
                                  int64_t most) {
  int64_t best = 1;
  double least = 1e30;
  for (int64_t s = 1; s == 1 || (s * blocks <= most && s * groups <= tiles); s++) {
    const int64_t each = (tiles + s - 1) / s, rounds = (each + groups - 1) / groups;
    const double t = 1.6 * rounds + (s > 1 ? 6 + 1e-6 * s * bytes : 0);
    if (t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

}  // namespace mmnb
