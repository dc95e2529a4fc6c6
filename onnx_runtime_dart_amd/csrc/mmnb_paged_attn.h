// Attention over a paged cache: the kernels and their launches, per cache type.
#pragma once

#include <algorithm>

#include "mmnb_paged_tile.h"

namespace mmnb {

// ---- who works on what
// The last entry of start[0 .. batch] at or below row t (rows' begins rise).  A wave narrows
// 65536 entries down in three rounds of loads.
__device__ __forceinline__ int seq_of_row_wave(const PagedArgs &a, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, span = a.batch + 1;  // the entry lies in [lo, lo + span)
  while (span > 1) {
    const int step = (span + 63) / 64, i = lo + lane * step;
    const bool below = lane * step < span && a.start[i] <= t;
    const int n = __popcll(__ballot(below));
    if (n == 0) return -1;
    span = min(step, lo + span - (lo + (n - 1) * step));
    lo += (n - 1) * step;
  }
  return a.start[lo] <= t ? lo : -1;
}
__device__ __forceinline__ int seq_of_row_lane(const PagedArgs &a, int t) {
  int lo = 0, hi = a.batch + 1;  // start[lo - 1] <= t < start[hi]
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.start[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1;
}

__device__ __forceinline__ int64_t uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// The sequences' shares of something in one line: share(b) each.  Sum over all of them, and the
// sequence that holds place x (with its first place).
template <typename F>
__device__ __forceinline__ int64_t line_length(int batch, F share) {
  int64_t sum = 0;
  for (int base = 0; base < batch; base += 64) {
    const int b = base + ((int)threadIdx.x & 63);
    sum += b < batch ? share(b) : 0;
  }
#pragma unroll
  for (int w = 1; w < 64; w *= 2) sum += __shfl_xor(sum, w);
  return uniform(sum);
}
template <typename F>
__device__ __forceinline__ int line_find(int batch, int64_t x, int64_t *first, F share) {
  int64_t before = 0;
  for (int base = 0; base < batch; base += 64) {
    const int lane = threadIdx.x & 63, b = base + lane;
    const int64_t n = b < batch ? share(b) : 0;
    int64_t upto = n;
#pragma unroll
    for (int w = 1; w < 64; w *= 2) {
      const int64_t y = __shfl_up(upto, w);
      upto += lane >= w ? y : 0;
    }
    const uint64_t past = __ballot(before + upto > x);
    if (past) {
      const int i = __builtin_ctzll(past);
      *first = before + uniform(__shfl(upto - n, i));
      return base + i;
    }
    before += uniform(__shfl(upto, 63));
  }
  return -1;
}
// First place of sequence b.
template <typename F>
__device__ __forceinline__ int64_t line_before(int b, F share) {
  return line_length(b, share);
}

__device__ __forceinline__ int two_of(const AttnArgs &t, int b) { return t.two ? t.two[b] : 0; }

template <int KT>
__device__ __forceinline__ PagedRange range_of(const PagedArgs &a, const AttnArgs &t, int b) {
  return paged_range(seq_of(a, b), t.window, two_of(t, b) - t.prefix, KT);
}

// Zero for a row that sees nothing, else the factor of its sums.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// A row again, as defined, where the matrix cores' sums were not finite.
template <typename T>
__device__ void redo_row(const PagedArgs &a, const AttnArgs &t, int b, const PagedSeq &s, int i,
                         int h) {
  const int lane = threadIdx.x & 63, row = s.row0 + i;
  RowState st = row_exact<T>(a, t, a.pages + b * a.cols, t.q + row * t.ldq + (int64_t)h * a.hd,
                             h, t.prefix + s.len - s.n + i, two_of(t, b), 0, t.prefix + s.len);
  float *o = t.out + row * t.ldo + (int64_t)h * a.hd;
  const bool none = st.l == 0.0f;
  if (lane < a.hd) o[lane] = none ? 0.0f : st.o0 / st.l;
  if (lane + 64 < a.hd) o[lane + 64] = none ? 0.0f : st.o1 / st.l;
}
// NaN for the rows of kv head g of a sequence that breaks the batch's promises.
__device__ __forceinline__ void refuse_rows(const PagedArgs &a, const AttnArgs &t,
                                            const PagedSeq &s, int g) {
  const int w = t.group * a.hd;
  for (int i = 0; i < s.n; i++)
    for (int d = threadIdx.x & 63; d < w; d += 64)
      t.out[(s.row0 + i) * t.ldo + (int64_t)g * w + d] = __builtin_nanf("");
}

// Partial results: sums o [hd] and (m, l) of each piece.
struct Pieces {
  float *o, *ml;
};
__device__ __forceinline__ void put_ml(const Pieces &p, int64_t i, float m, float l) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  *(f2 *)(p.ml + 2 * i) = f2{m, l};
}

// ---------------------------------------------------------------------------
// Few rows of a sequence and kv head (up to MF): one stream of keys and values, bound by
// memory.  All tiles of all sequences and heads lie in one line that is dealt to the waves in
// equal runs, so that no wave waits for the longest sequence; a wave has its own stages in LDS
// and never meets another.  Rows whose keys lie in several waves' runs are merged by
// k_paged_merge.
// ---------------------------------------------------------------------------
struct TokenPlan {
  int least;      // tiles of a wave, if there are so many
  int waves;      // most
  bool keep;      // all rows are merged with more pieces
  Pieces out;
};
// Slot (of MF rows) of the piece that wave w has of pair x of sequence and head: with every
// piece kept one of waves + pairs, else, with the whole rows stored at once, one of two a wave.
__device__ __forceinline__ int64_t token_slot(bool keep, int64_t w, int64_t x, bool first) {
  return keep ? w + x : 2 * w + first;
}

// Waves of a workgroup, and workgroups of a CU, with two stages of keys and values each in the
// CU's 160 KB.
template <typename T, int HD>
struct TokenShape {
  static constexpr int kStage = 2 * kPagedTokenTile * Row<T, HD>::kBytes;
  static constexpr int kWaves = kStage <= 16384 ? 4 : 2;
  static constexpr int kLds = kWaves * 2 * kStage;
  static constexpr int kPerCu = 160 * 1024 / kLds;
};

template <typename T, int HD, int MF>
__global__ void __launch_bounds__((64 * TokenShape<T, HD>::kWaves)) k_paged_token(PagedArgs a, AttnArgs t, TokenPlan pl) {
  constexpr int KT = kPagedTokenTile;
  typedef WaveRows<T, HD, MF, KT> W;
  typedef Loader<T, HD, KT> L;
  constexpr int kTile = KT * Row<T, HD>::kBytes, kStage = 2 * kTile;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char *mine = smem + wave * 2 * kStage;
  L load;
  load.begin(a, 0, 1);
  const int G = a.kv_heads;
  auto share = [&](int b) { return (int64_t)range_of<KT>(a, t, b).n * G; };
  const int64_t total = line_length(a.batch, share);
  if (total == 0) return;
  const int64_t workers = paged_workers(total, pl.waves, pl.least);
  const int64_t w = (int64_t)wave * gridDim.x + blockIdx.x;  // neighbours on different CUs
  if (w >= workers) return;
  int64_t x = paged_first(total, w, workers), before = 0;
  const int64_t xe = paged_first(total, w + 1, workers);
  if (x >= xe) return;
  int b = line_find(a.batch, x, &before, share);
  W r;
  while (true) {
    const PagedSeq s = seq_of(a, b);
    const int two = two_of(t, b);
    const PagedRange rg = paged_range(s, t.window, two - t.prefix, KT);
    const int g = (int)((x - before) / rg.n);
    const int t0 = (int)(x - before - (int64_t)g * rg.n);
    const int t1 = (int)min((int64_t)rg.n, t0 + (xe - x));
    if (s.bad) {
      if (!pl.keep) refuse_rows(a, t, s, g);
    } else {
      const int c = lane % MF, i = c / t.group, h = g * t.group + c % t.group;
      const bool live = i < s.n;
      r.begin(t, live ? t.q + (s.row0 + i) * t.ldq + (int64_t)h * a.hd : nullptr, a.hd, h,
              t.prefix + s.len - s.n + i, two);
      const int32_t *table = a.pages + b * a.cols;
      const int64_t head = g * a.sh;
      PageIds ids;
      bool bad = false;
      auto issue = [&](int k) {
        const int j = rg.lo + k * KT;
        ids.cover(a, table, j, s.len);
        bad = bad || ids.bad;
        char *st = mine + (k & 1) * kStage;
        load.tile(a, ids, head, j, s.len - 1, 0, 1, st, st + kTile);
      };
      issue(t0);
      for (int k = t0; k < t1; k++) {
        if (k + 1 < t1) {
          issue(k + 1);
          wait_dma<L::per_wave(1)>();
        } else {
          wait_dma<0>();
        }
        const int jp = t.prefix + rg.lo + k * KT;
        const char *st = mine + (k & 1) * kStage;
        if (r.any(jp, t.window)) r.tile(t, st, st + kTile, jp, t.prefix + s.len);
        asm volatile("" ::: "memory");  // the stage is read before it is filled again
      }
      const bool fine = r.end() && !bad;
      if (t0 == 0 && t1 == rg.n && !pl.keep) {
        if (live && fine)
          r.store(t.out + (s.row0 + i) * t.ldo + (int64_t)h * a.hd, a.hd, inverse(r.l));
        uint64_t again = __ballot(live && !fine && lane < MF);
        while (again) {
          const int k = __builtin_ctzll(again);
          again &= again - 1;
          redo_row<T>(a, t, b, s, k / t.group, g * t.group + k % t.group);
        }
      } else if (live) {
        const int64_t slot =
            token_slot(pl.keep, w, (int64_t)b * G + g, t0 == 0) * MF + c;
        r.store(pl.out.o + slot * a.hd, a.hd, 1.0f);
        if (lane < MF) put_ml(pl.out, slot, r.m, fine ? r.l : __builtin_nanf(""));
      }
    }
    x += t1 - t0;
    if (x >= xe) return;
    if (x - before >= (int64_t)rg.n * G) {  // x is a place of the next sequence that has any
      before += (int64_t)rg.n * G;
      do b++;
      while (share(b) == 0);
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup's four waves, 32 rows each, share the tiles of their kv head, which
// costs every tile's bytes once for 128 rows.  Bound by the matrix cores and the exponentials.
// Row k of a sequence's rows and a head's group is row k / group of query head k % group.
// ---------------------------------------------------------------------------
struct PromptPlan {
  int splits;     // parts of the keys; with more than one, or with keep, results are pieces
  bool keep;
  bool prefix;    // rows of all sequences over the shared prefix alone
  Pieces out;     // [splits][tokens][heads]
};

template <typename T, int HD>
__global__ void __launch_bounds__(256, 2) k_paged_prompt(PagedArgs a, AttnArgs t, PromptPlan pl) {
  constexpr int KT = sizeof(T) == 2 ? 64 : 32, MF = 32;
  typedef WaveRows<T, HD, MF, KT> W;
  typedef Loader<T, HD, KT> L;
  constexpr int kTile = KT * Row<T, HD>::kBytes, kStage = 2 * kTile;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x, R = t.group;
  const int place = gridDim.y - 1 - blockIdx.y;  // long rows first
  int b = 0, tile = place, rows = a.tokens * R, two = 0;
  PagedSeq s = {0, a.tokens, 0, false};
  if (!pl.prefix) {
    int64_t before = 0;
    b = line_find(a.batch, place, &before, [&](int i) {
      const PagedSeq q = seq_of(a, i);
      return (int64_t)(q.n == 0 ? 0
                       : q.bad  ? 1
                                : (q.n * R + kPagedPromptRows - 1) / kPagedPromptRows);
    });
    if (b < 0) return;
    tile = place - (int)before;
    s = seq_of(a, b);
    two = two_of(t, b);
    rows = s.n * R;
    if (s.bad) {
      if (blockIdx.z == 0 && wave == 0 && pl.splits == 1) refuse_rows(a, t, s, g);
      return;
    }
  }
  L load;
  load.begin(a, wave, 4);
  const int first = tile * kPagedPromptRows, c = lane % MF, k = first + wave * MF + c;
  const bool live = k < rows;
  const int i = k / R, h = g * R + k % R, row = s.row0 + i;
  int pos = t.prefix + s.len - s.n + i, mine2 = two;
  if (pl.prefix) {
    pos = t.prefix;  // past all of the prefix
    mine2 = 0;
    if (live && (t.window || t.slopes || t.two)) {
      const int q = seq_of_row_lane(a, row);
      if (q >= 0 && q < a.batch) {
        const PagedSeq u = seq_of(a, q);
        pos = u.bad ? t.prefix : t.prefix + u.len - u.n + (row - u.row0);
        mine2 = two_of(t, q);
      }
    }
  }
  W r;
  r.begin(t, live ? t.q + row * t.ldq + (int64_t)h * a.hd : nullptr, a.hd, h, pos, mine2);
  // tiles of the prefix, then of the sequence's own keys, up to the last that a row sees
  const int p0 = t.prefix + s.len - s.n + first / R;
  const int p1 = min(t.prefix + s.len - 1,
                     t.prefix + s.len - s.n + (first + kPagedPromptRows - 1) / R);
  const int from = t.window && two <= 0 && !pl.prefix ? max(0, p0 - t.window + 1) : 0;
  const int own = pl.prefix ? 0 : min(s.len, max(p1 + 1, two) - t.prefix);
  const int loa = min(from, t.prefix) / KT * KT, lob = max(0, from - t.prefix) / KT * KT;
  const int na = (t.prefix - loa + KT - 1) / KT, nb = own > lob ? (own - lob + KT - 1) / KT : 0;
  const int z = blockIdx.z;
  const int k0 = (int)paged_first(na + nb, z, pl.splits);
  const int k1 = (int)paged_first(na + nb, z + 1, pl.splits);
  const int32_t *table = a.pages + b * a.cols;
  const int64_t head = g * a.sh;
  PageIds ids;
  bool bad = false;
  auto issue = [&](int n) {
    const bool pre = n < na;
    const int j = pre ? loa + n * KT : lob + (n - na) * KT, end = pre ? t.prefix : own;
    ids.cover(a, pre ? t.ppages : table, j, end);
    bad = bad || ids.bad;
    char *st = smem + (n & 1) * kStage;
    load.tile(a, ids, head, j, end - 1, wave, 4, st, st + kTile);
  };
  if (k0 < k1) issue(k0);
  for (int n = k0; n < k1; n++) {
    if (n + 1 < k1) {
      issue(n + 1);
      wait_dma<L::per_wave(4)>();
    } else {
      wait_dma<0>();
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const bool pre = n < na;
    const int jp = pre ? loa + n * KT : t.prefix + lob + (n - na) * KT;
    const char *st = smem + (n & 1) * kStage;
    if (r.any(jp, t.window)) r.tile(t, st, st + kTile, jp, t.prefix + (pre ? 0 : own));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
  }
  const bool fine = r.end() && !bad;
  if (pl.splits == 1 && !pl.keep) {
    if (live && fine) r.store(t.out + row * t.ldo + (int64_t)h * a.hd, a.hd, inverse(r.l));
    uint64_t again = __ballot(live && !fine && lane < MF);
    while (again) {
      const int u = __builtin_ctzll(again);
      again &= again - 1;
      const int kk = first + wave * MF + u;
      redo_row<T>(a, t, b, s, kk / R, g * R + kk % R);
    }
  } else if (live) {
    const int64_t slot = ((int64_t)z * a.tokens + row) * t.heads + h;
    r.store(pl.out.o + slot * a.hd, a.hd, 1.0f);
    if (lane < MF) put_ml(pl.out, slot, r.m, fine ? r.l : __builtin_nanf(""));
  }
}

// ---------------------------------------------------------------------------
// Rows from their pieces, in the pieces' order, a wave per row and head.
// ---------------------------------------------------------------------------
struct MergePlan {
  TokenPlan token;    // token.waves: 0 without them
  int mf;
  int splits;         // of PromptPlan's pieces; 0 without them
  Pieces split;
};

// Adds n pieces, at slots at(0) .. at(n - 1), to a row's state.
template <typename F>
__device__ __forceinline__ void add_pieces(RowState &s, const Pieces &p, int64_t n, int hd,
                                           F at) {
  const int lane = threadIdx.x & 63;
  for (int64_t base = 0; base < n; base += 64) {
    const int cnt = (int)min((int64_t)64, n - base);
    const int64_t slot = at(base + min(lane, cnt - 1));
    const float m = lane < cnt ? p.ml[2 * slot] : kNegInf;
    const float l = lane < cnt ? p.ml[2 * slot + 1] : 0.0f;
    float top = m;
#pragma unroll
    for (int w = 1; w < 64; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
    const float next = fmaxf(s.m, top), ref = next == kNegInf ? 0.0f : next;
    const float old = __builtin_amdgcn_exp2f(s.m - ref);
    const float f = __builtin_amdgcn_exp2f(m - ref);
    float sum = l * f;
#pragma unroll
    for (int w = 1; w < 64; w *= 2) sum += __shfl_xor(sum, w);
    s.m = next;
    s.l = s.l * old + sum;
    s.o0 *= old;
    s.o1 *= old;
#pragma unroll 4
    for (int i = 0; i < cnt; i++) {
      const float *o = p.o + __shfl(slot, i) * hd;
      const float g = __shfl(f, i);
      if (lane < hd) s.o0 = fmaf(g, o[lane], s.o0);
      if (lane + 64 < hd) s.o1 = fmaf(g, o[lane + 64], s.o1);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_paged_merge(PagedArgs a, AttnArgs t, MergePlan pl) {
  constexpr int KT = kPagedTokenTile;
  const int64_t rh =
      (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = (int)(rh / t.heads), h = (int)(rh % t.heads), lane = threadIdx.x & 63;
  if (row >= a.tokens) return;
  const int b = __builtin_amdgcn_readfirstlane(seq_of_row_wave(a, row));
  if (b < 0 || b >= a.batch) return;
  const PagedSeq s = seq_of(a, b);
  const int i = row - s.row0, g = h / t.group, G = a.kv_heads;
  float *o = t.out + row * t.ldo + (int64_t)h * a.hd;
  if (s.bad) {
    if (lane < a.hd) o[lane] = __builtin_nanf("");
    if (lane + 64 < a.hd) o[lane + 64] = __builtin_nanf("");
    return;
  }
  if (i >= s.n) return;
  RowState st = {kNegInf, 0.0f, 0.0f, 0.0f};
  if (pl.splits)
    add_pieces(st, pl.split, pl.splits, a.hd,
               [&](int64_t z) { return (z * a.tokens + row) * t.heads + h; });
  if (pl.token.waves) {
    auto share = [&](int q) { return (int64_t)range_of<KT>(a, t, q).n * G; };
    const int64_t total = line_length(a.batch, share), before = line_before(b, share);
    const int64_t workers = paged_workers(total, pl.token.waves, pl.token.least);
    const int n = range_of<KT>(a, t, b).n;
    const int64_t x0 = before + (int64_t)g * n, x1 = x0 + n - 1;
    const int64_t w0 = paged_worker_of(total, x0, workers);
    const int64_t w1 = paged_worker_of(total, x1, workers);
    if (w0 == w1 && !pl.token.keep) return;  // stored by its wave
    const int c = i * t.group + h % t.group;
    add_pieces(st, pl.token.out, w1 - w0 + 1, a.hd, [&](int64_t k) {
      return token_slot(pl.token.keep, w0 + k, (int64_t)b * G + g, k == 0) * pl.mf + c;
    });
  }
  const bool fine = paged_finite(st.l) && paged_finite(st.o0) && paged_finite(st.o1);
  if (!__all(fine)) {
    redo_row<T>(a, t, b, s, i, h);
    return;
  }
  const float f = inverse(st.l);
  if (lane < a.hd) o[lane] = st.o0 * f;
  if (lane + 64 < a.hd) o[lane + 64] = st.o1 * f;
}

// ---------------------------------------------------------------------------
// Attention, a wave per row and head: caches whose rows lie too far apart for a tile's loads.
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) k_paged_rows(PagedArgs a, AttnArgs t) {
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = (int)(r / t.heads), h = (int)(r % t.heads), lane = threadIdx.x & 63;
  if (row >= a.tokens) return;
  const int b = __builtin_amdgcn_readfirstlane(seq_of_row_wave(a, row));
  if (b < 0 || b >= a.batch) return;
  const PagedSeq s = seq_of(a, b);
  if (s.bad) {
    float *o = t.out + row * t.ldo + (int64_t)h * a.hd;
    if (lane < a.hd) o[lane] = __builtin_nanf("");
    if (lane + 64 < a.hd) o[lane + 64] = __builtin_nanf("");
  } else if (row < s.row0 + s.n) {
    redo_row<T>(a, t, b, s, row - s.row0, h);
  }
}

// ---- launches
template <typename K>
int allow_lds(K kern, size_t bytes) {
  if (bytes > 65536) {
    const hipError_t e = hipFuncSetAttribute(
        (const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) return check_hip(e, "hipFuncSetAttribute");
  }
  return MMNB_OK;
}

template <typename T, int HD, int MF>
int launch_token(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t, const TokenPlan &pl) {
  typedef TokenShape<T, HD> S;
  auto kern = k_paged_token<T, HD, MF>;
  if (int rc = allow_lds(kern, S::kLds)) return rc;
  return launch(ctx, kKernPagedAttn, kern, dim3((unsigned)(pl.waves / S::kWaves)),
                dim3(64 * S::kWaves), S::kLds, a, t, pl);
}
template <typename T, int HD>
int launch_prompt(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t, const PromptPlan &pl,
                  int64_t tiles) {
  const size_t lds = 4 * (sizeof(T) == 2 ? 64 : 32) * Row<T, HD>::kBytes;
  auto kern = k_paged_prompt<T, HD>;
  if (int rc = allow_lds(kern, lds)) return rc;
  return launch(ctx, kKernPagedAttn, kern,
                dim3((unsigned)a.kv_heads, (unsigned)tiles, (unsigned)pl.splits), dim3(256), lds,
                a, t, pl);
}

template <typename T, int HD>
int launch_attention(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t) {
  const int64_t rows = (int64_t)a.max_q * t.group, all = (int64_t)a.tokens * t.heads;
  const int cus = ctx->cu_count;
  const bool token = rows <= kPagedTokenRows, prefix = token && t.prefix > 0;
  MergePlan mp = {};
  mp.mf = rows <= 16 ? 16 : 32;
  PromptPlan pp = {};
  pp.splits = 1;
  int64_t tiles = 0, slots = 0;
  if (token) {
    mp.token.waves = cus * TokenShape<T, HD>::kPerCu * TokenShape<T, HD>::kWaves;
    mp.token.least = 2;
    mp.token.keep = prefix;
    slots = mp.mf * (prefix ? mp.token.waves + (int64_t)a.batch * a.kv_heads
                            : 2 * (int64_t)mp.token.waves);
  }
  if (!token || prefix) {
    const int kt = sizeof(T) == 2 ? 64 : 32;
    const int64_t keys = (prefix ? t.prefix : (int64_t)t.prefix + a.max_kv);
    tiles = prefix ? ((int64_t)a.tokens * t.group + kPagedPromptRows - 1) / kPagedPromptRows
                   : paged_row_tiles(a.batch, a.tokens, a.max_q, t.group);
    pp.splits = (int)paged_splits(tiles * a.kv_heads, (keys + kt - 1) / kt, cus);
    pp.keep = pp.prefix = prefix;
    if (pp.splits > 1 || prefix) mp.splits = pp.splits;
  }
  const int64_t total = slots + mp.splits * all;
  if (total) {
    void *buf = nullptr;
    const size_t need = (size_t)total * (a.hd + 2) * 4;
    if (int rc = scratch_get(ctx, kPagedScratch, std::max(need, kPagedScratchBytes), &buf))
      return rc;
    mp.token.out.o = (float *)buf;
    mp.split.o = mp.token.out.o + slots * a.hd;
    mp.token.out.ml = mp.split.o + mp.splits * all * a.hd;
    mp.split.ml = mp.token.out.ml + 2 * slots;
    pp.out = mp.split;
  }
  if (!token || prefix)
    if (int rc = launch_prompt<T, HD>(ctx, a, t, pp, tiles)) return rc;
  if (token) {
    const int rc = mp.mf == 16 ? launch_token<T, HD, 16>(ctx, a, t, mp.token)
                               : launch_token<T, HD, 32>(ctx, a, t, mp.token);
    if (rc) return rc;
  }
  if (!total) return MMNB_OK;
  return launch(ctx, kKernPagedMerge, k_paged_merge<T>, dim3((unsigned)((all + 3) / 4)),
                dim3(256), 0, a, t, mp);
}

template <typename T>
int paged_attention(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t) {
  // a tile's loads reach eight rows with 31 bits of offset
  if (a.sr > (1 << 23))
    return launch(ctx, kKernPagedAttn, k_paged_rows<T>,
                  dim3((unsigned)(((int64_t)a.tokens * t.heads + 3) / 4)), dim3(256), 0, a, t);
  if (a.hd <= 64) return launch_attention<T, 64>(ctx, a, t);
  if (a.hd <= 96) return launch_attention<T, 96>(ctx, a, t);
  return launch_attention<T, 128>(ctx, a, t);
}

}  // namespace mmnb
