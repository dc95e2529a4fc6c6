// Attention over a paged cache: the kernels and their launches, per cache type.
#pragma once

#include <algorithm>

#include "mmnb_paged_tile.h"

namespace mmnb {

// ---- who works on what
// The last entry of start[0 .. batch] at or below row t (-1: none), the row's sequence where starts
// rise; else any.  A wave narrows 65536 entries down in three rounds of loads.
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
// The sequence that holds row t, by a lane for itself (-1: none that a search of rising starts
// finds).
__device__ __forceinline__ int seq_of_row_lane(const PagedArgs &a, int t) {
  int lo = 0, hi = a.batch + 1;  // start[lo - 1] <= t < start[hi]
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.start[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  lo--;
  return lo >= 0 && lo < a.batch && paged_holds(a.start, lo, t) ? lo : -1;
}

__device__ __forceinline__ int two_of(const AttnArgs &t, int b) {
  return t.two ? max(0, t.two[b]) : 0;
}

// Inclusive sums over the wave's lanes.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31
  return x;
}

// The batch's sequences, 64 at a time in a wave's lanes, so that a batch of up to 64 costs one
// round of loads however often it is looked at.  Every sequence has a share of a line (share(s,
// r): its places, all of them together below 2^31).
struct Seqs {
  int base = -1;
  PagedSeq s = {0, 0, 0, false};   // of sequence base + lane
  PagedRange r = {0, 0};
  int two = 0;

  template <int KT>
  __device__ __forceinline__ void look(const PagedArgs &a, const AttnArgs &t, int b) {
    const int want = b & ~63;
    if (want == base) return;
    base = want;
    const int i = want + ((int)threadIdx.x & 63);
    s = {0, 0, 0, false};
    r = {0, 0};
    two = 0;
    if (i < a.batch) {
      two = two_of(t, i);
      s = seq_of(a, i);
      r = paged_range(s, t.window, two - t.prefix, KT);
    }
  }
  __device__ __forceinline__ PagedSeq seq(int b) const {
    const int i = b & 63;
    return {__builtin_amdgcn_readlane(s.row0, i), __builtin_amdgcn_readlane(s.n, i),
            __builtin_amdgcn_readlane(s.len, i), __builtin_amdgcn_readlane((int)s.bad, i) != 0};
  }
  __device__ __forceinline__ PagedRange range(int b) const {
    return {__builtin_amdgcn_readlane(r.lo, b & 63), __builtin_amdgcn_readlane(r.n, b & 63)};
  }
  __device__ __forceinline__ int two_way(int b) const {
    return __builtin_amdgcn_readlane(two, b & 63);
  }
  // The line's length, and the places before sequence b.
  template <int KT, typename F>
  __device__ __forceinline__ int length(const PagedArgs &a, const AttnArgs &t, F share, int b,
                                        int *before) {
    int sum = 0, first = 0;
    for (int c = (a.batch - 1) & ~63; c >= 0; c -= 64) {
      look<KT>(a, t, c);
      const int x = share(s, r), upto = wave_scan(x), all = __builtin_amdgcn_readlane(upto, 63);
      sum += all;
      if (c == (b & ~63)) first += __builtin_amdgcn_readlane(upto - x, b & 63);
      else if (c < b) first += all;
    }
    *before = first;
    return sum;
  }
  // The sequence that holds place x, and the places before it (-1 behind the last).
  template <int KT, typename F>
  __device__ __forceinline__ int find(const PagedArgs &a, const AttnArgs &t, F share, int x,
                                      int *before) {
    int done = 0;
    for (int c = 0; c < a.batch; c += 64) {
      look<KT>(a, t, c);
      const int n = share(s, r), upto = wave_scan(n);
      const uint64_t past = __ballot(done + upto > x);
      if (past) {
        const int i = __builtin_ctzll(past);
        *before = done + __builtin_amdgcn_readlane(upto - n, i);
        return c + i;
      }
      done += __builtin_amdgcn_readlane(upto, 63);
    }
    return -1;
  }
};

// Zero for a row that sees nothing, else the factor of its sums.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// A row again, as defined, where the matrix cores' sums were not finite.
template <typename T>
__device__ void redo_row(const PagedArgs &a, const AttnArgs &t, int b, const PagedSeq &s, int i,
                         int h) {
  const int lane = threadIdx.x & 63, row = s.row0 + i, p = t.prefix + s.len - s.n + i;
  const int two = two_of(t, b);
  const PagedSpan keys = paged_row_span(p, t.window, two, t.prefix + s.len);
  RowState st = row_exact<T>(a, t, a.pages + b * a.cols, t.q + row * t.ldq + (int64_t)h * a.hd,
                             h, p, two, keys.lo, keys.hi);
  float *o = t.out + row * t.ldo + (int64_t)h * a.hd;
  const bool none = st.l == 0.0f;
  if (lane < a.hd) o[lane] = none ? 0.0f : st.o0 / st.l;
  if (lane + 64 < a.hd) o[lane + 64] = none ? 0.0f : st.o1 / st.l;
}
// The same for row `row` of the call, by a wave that looks for its sequence (nothing for a row
// that has none).
template <typename T>
__device__ __forceinline__ void row_anew(const PagedArgs &a, const AttnArgs &t, int row, int h) {
  const int b = scan_for_row(a, row), lane = threadIdx.x & 63;
  if (b < 0) return;
  const PagedSeq s = seq_of(a, b);
  if (!s.bad) {
    redo_row<T>(a, t, b, s, row - s.row0, h);
    return;
  }
  float *o = t.out + row * t.ldo + (int64_t)h * a.hd;
  if (lane < a.hd) o[lane] = __builtin_nanf("");
  if (lane + 64 < a.hd) o[lane + 64] = __builtin_nanf("");
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
// k_paged_merge.  Single tokens of 64 sequences of up to 8192 keys, 32 heads on 8 of 128 bf16
// (1.22 GB, all of it fetched): 223 us with the merge, 5.5 TB/s, where a large copy, half of it
// writes, reaches 4.7; of two of up to 131071 keys on fp16 137 us.  Small calls are bound by latency: 523 keys of one sequence, 16
// heads on 8, take 9 us and the merge 5, about 2000 cycles for each load that needs another's
// result.  (Merging in the same launch, by the wave that completes a row, took as long: 14.4 us
// in all, and 222 instead of 190 behind a prefix of 32768 keys.)
// ---------------------------------------------------------------------------
struct TokenPlan {
  int waves;      // most that take part
  bool keep;      // all rows are merged with more pieces
  bool whole;     // a sequence and head is one place of the line, and never cut
  int flat;       // tiles of the prefix's keys (0: none), which with each of `sets` sets of MF
  int sets;       // rows of the whole call lie in the line before the sequences'
  Pieces out;
};
// Slot (of MF rows) of the piece that wave w has of pair x of sequence and head: with every
// piece kept one of waves + pairs, else, with the whole rows stored at once, one of two a wave.
__device__ __forceinline__ int64_t token_slot(bool keep, int w, int64_t x, bool first) {
  return keep ? w + x : 2 * (int64_t)w + first;
}

// Waves of a workgroup, and workgroups of a CU, with two stages of keys and values each in the
// CU's 160 KB: up to 128 KB of loads in flight, of which 35 would cover the latency.
template <typename T, int HD>
struct TokenShape {
  static constexpr int kStage = 2 * kPagedTokenTile * Row<T, HD, 32>::kBytes;
  static constexpr int kWaves = kStage <= 16384 ? 4 : 2;
  static constexpr int kLds = kWaves * 2 * kStage;
  static constexpr int kPerCu = 160 * 1024 / kLds;
};

// A wave's rows over the shared prefix: the lane's row of the call, whatever its sequence.  The
// rows see all of it; their places count only with a window or slopes.
template <typename W>
__device__ __forceinline__ void begin_prefix(W &r, const PagedArgs &a, const AttnArgs &t,
                                             typename W::Query &y, bool live, int row) {
  if (!t.window && !t.slopes) {
    r.begin(t, y, live ? t.prefix : -1, 0, t.prefix, t.prefix, 0, 0);
    return;
  }
  int pos = t.prefix, own = 0;
  if (live) {
    const int q = seq_of_row_lane(a, row);
    if (q >= 0) {
      const PagedSeq u = seq_of(a, q);
      pos = u.bad ? t.prefix : t.prefix + u.len - u.n + (row - u.row0);
      own = two_of(t, q);
    } else {
      y.x[0][0] = __builtin_nanf("");  // no sequence's, or k_paged_merge finds it and starts anew
    }
  }
  r.begin_any(t, y, live, pos, own);
}

template <typename T, int HD, int MF>
__global__ void __launch_bounds__((64 * TokenShape<T, HD>::kWaves))
k_paged_token(PagedArgs a, AttnArgs t, TokenPlan pl) {
  constexpr int KT = kPagedTokenTile;
  typedef WaveRows<T, HD, MF, KT, true> W;
  typedef Loader<T, HD, MF, KT> L;
  constexpr int kTile = KT * Row<T, HD, 32>::kBytes, kStage = 2 * kTile;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char *mine = smem + wave * 2 * kStage;
  L load;
  load.begin(a);
  const int G = a.kv_heads, R = t.group;
  auto share = [&](const PagedSeq &, const PagedRange &r) {
    return pl.whole ? (r.n ? G : 0) : r.n * G;
  };
  Seqs seqs;
  int before;
  const int lead = pl.flat * pl.sets * G;  // places of the prefix
  const int total = lead + seqs.length<KT>(a, t, share, 0, &before);
  const int each = paged_each(total, pl.waves);
  const int w = wave * gridDim.x + blockIdx.x;  // neighbours on different CUs
  if ((int64_t)w * each >= total) return;
  int x = w * each;
  const int xe = min(total, x + each);
  int b = -1;
  before = 0;
  if (x >= lead) {
    b = seqs.find<KT>(a, t, share, x - lead, &before);
    before += lead;
  }
  const int c = lane % MF;
  W r;
  while (true) {
    const bool pre = x < lead;  // of the prefix, with the rows of all sequences
    const PagedSeq s = pre ? PagedSeq{0, a.tokens, t.prefix, false} : seqs.seq(b);
    const PagedRange rg = pre ? PagedRange{t.seen, pl.flat} : seqs.range(b);
    const int two = pre ? 0 : seqs.two_way(b);
    const int places = pl.whole ? 1 : rg.n;
    const int pair = (uint32_t)(x - before) / (uint32_t)places;
    const int t0 = x - before - pair * places, t1 = pl.whole ? rg.n : min(rg.n, t0 + (xe - x));
    int g = pair, r0 = 0;
    if (pre) {
      g = (uint32_t)pair / (uint32_t)pl.sets;
      r0 = (pair - g * pl.sets) * MF;
    }
    if (s.bad) {
      if (!pl.keep) refuse_rows(a, t, s, g);
    } else {
      const GroupRow me = group_row(t, r0 + c);
      const int i = me.i, h = g * R + me.r;
      const bool live = i < s.n;
      const int32_t *table = pre ? t.ppages : a.pages + b * a.cols;
      const int64_t head = g * a.sh;
      PageIds ids;
      auto issue = [&](int k) {
        const int j = rg.lo + k * KT;
        ids.cover(a, table, j, s.len, pre ? 0 : t.prefix);
        char *st = mine + (k & 1) * kStage;
        load.tile(a, ids, head, j, s.len - 1, 0, 1, st, st + kTile);
      };
      // the queries' loads, the page numbers' and the first tile's: two round trips
      typename W::Query y;
      W::load(y, t, live ? t.q + (s.row0 + i) * t.ldq + (int64_t)h * a.hd : nullptr, a.hd, h);
      issue(t0);
      if (pre) {
        begin_prefix(r, a, t, y, live, i);
      } else {
        const int p0 = t.prefix + s.len - s.n;
        r.begin(t, y, live ? p0 + i : -1, live ? two : 0, p0, p0 + s.n - 1, two, two);
      }
      const int off = pre ? 0 : t.prefix;
      for (int k = t0; k < t1; k++) {
        if (k + 1 < t1) {
          issue(k + 1);
          wait_dma<L::per_wave(1)>();
        } else {
          wait_dma<0>();
        }
        const int jp = off + rg.lo + k * KT;
        const char *st = mine + (k & 1) * kStage;
        if (r.any(jp, t.window)) r.tile(t, st, st + kTile, jp, off + s.len);
        asm volatile("" ::: "memory");  // the stage is read before it is filled again
      }
      const bool fine = r.end() && !ids.missed(a, t, r);
      if (t0 == 0 && t1 == rg.n && !pl.keep) {
        if (live && fine)
          r.store(t.out + (s.row0 + i) * t.ldo + (int64_t)h * a.hd, a.hd, inverse(r.l));
        uint64_t again = __ballot(live && !fine && lane < MF);
        while (again) {
          const int k = __builtin_ctzll(again);
          again &= again - 1;
          redo_row<T>(a, t, b, s, k / R, g * R + k % R);
        }
      } else if (live) {
        const int64_t at = pre ? pair : pl.sets * G + (int64_t)b * G + g;
        const int64_t slot = token_slot(pl.keep, w, at, t0 == 0) * MF + c;
        r.store(pl.out.o + slot * a.hd, a.hd, 1.0f);
        if (lane < MF) put_ml(pl.out, slot, r.m, fine ? r.l : __builtin_nanf(""));
      }
    }
    x += pl.whole ? 1 : t1 - t0;
    if (x >= xe) return;
    if (pre ? x >= lead : x - before >= places * G) {  // a place of the next sequence that has any
      before = x;
      do seqs.look<KT>(a, t, ++b);
      while (seqs.range(b).n == 0);
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup's four waves, 32 rows each, share the tiles of their kv head, which
// costs every tile's bytes once for 128 rows.  Bound by the matrix cores and the exponentials.
// Row k of a sequence's rows and a head's group is row k / group of query head k % group.
// Where workgroups are few, NG = 2 groups of four waves take a tile each in turn, with stages of
// their own, and the second's sums are added to the first's at the end.
// 8192 rows of one sequence, 32 heads on 8 of 128 fp16: 0.96 ms, 1.15 PFLOP/s of products with
// both terms counted, where a library product of 8192^3 reaches 1.08.  The matrix cores are busy
// for 64% of the cycles, and the clock falls to 1.8 GHz: cycles saved come back as time by half
// (17% fewer when the reads lost their bank conflicts, 8% less time).  A unit of keys and a
// step's values are read from LDS before the products of the one before, whose time hides them:
// 1016 -> 956 us; one barrier a tile and reads without conflicts: 935.
// (Equal runs of all tiles' keys dealt to two workgroups a CU balance better but leave every
// row in pieces: 169 us for the uneven prompts, which take 140 whole.)
// ---------------------------------------------------------------------------
template <typename T, int HD, int MF, int NG>
struct Prompt {
  // (three terms of 128 values leave no registers for 32 rows' scores of 64 keys)
  static constexpr int KT =
      sizeof(T) == 4 || (Operand<T>::kTerms == 3 && HD == 128 && MF == 32) ? 32 : 64;
  static constexpr int kRows = 4 * MF, kThreads = 256 * NG;
  static constexpr int kPerCu = 2 / NG;  // workgroups of a CU, eight waves
  typedef WaveRows<T, HD, MF, KT, false> W;
  typedef Loader<T, HD, MF, KT> L;
  static constexpr int kTile = KT * Row<T, HD, 32>::kBytes, kStage = 2 * kTile;
  static constexpr int kLds = NG * 2 * kStage;
  static_assert(NG == 1 || 4 * W::kPutBytes <= kLds, "");

  // Tiles [k0, k1) of `keys`, all of them in the first group's rows; false in a group that has
  // given its sums away.  A bad page that they see makes the sums NaN.
  static __device__ __forceinline__ bool run(const PagedArgs &a, const AttnArgs &t, W &r,
                                             const L &load, char *smem, const int32_t *table,
                                             int64_t head, const PagedKeys &keys, int k0,
                                             int k1) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % 4;
    const int group = NG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    char *mine = smem + group * 2 * kStage;
    PageIds ids;
    auto issue = [&](int n, int stage) {
      const bool pre = n < keys.na;
      const int j = pre ? keys.loa + n * KT : keys.lob + (n - keys.na) * KT;
      const int end = pre ? t.prefix : keys.own;
      ids.cover(a, pre ? t.ppages : table, j, end, pre ? 0 : t.prefix);
      char *st = mine + stage * kStage;
      load.tile(a, ids, head, j, end - 1, wave, 4, st, st + kTile);
    };
    int n = k0 + group;
    if (n < k1) issue(n, 0);
    const int rounds = (k1 - k0 + NG - 1) / NG;
    for (int m = 0; m < rounds; m++, n += NG) {
      wait_dma<0>();
      barrier();  // the round's tiles are there, and the stages of the last one read
      if (n + NG < k1) issue(n + NG, (m + 1) & 1);
      const bool pre = n < keys.na;
      const int jp = pre ? keys.loa + n * KT : t.prefix + keys.lob + (n - keys.na) * KT;
      const char *st = mine + (m & 1) * kStage;
      if (n < k1 && r.any(jp, t.window))
        r.tile(t, st, st + kTile, jp, t.prefix + (pre ? 0 : keys.own));
    }
    if (ids.missed(a, t, r)) r.l = __builtin_nanf("");
    if constexpr (NG == 2) {
      barrier();
      if (group == 1) r.put(smem + wave * W::kPutBytes);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      barrier();
      if (group == 1) return false;
      r.add(smem + wave * W::kPutBytes);
    }
    return true;
  }
  static __device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

// Rows of all sequences over the shared prefix alone, whose keys they all see but for a window:
// pieces [splits][tokens][heads] of `blocks` workgroups for each part.  The `beside` workgroups
// before them take the sequences' own keys, where these are few: memory's work beside the matrix
// cores', in one launch.
struct PrefixPlan {
  int splits, blocks, beside;
  Pieces out;
  Pieces own;     // [batch][kv_heads][kBesideRows]
};
constexpr int kBesideRows = 16;   // most rows of a sequence and kv head
// Most tiles of a sequence's own keys, which one wave takes after each other, about 2.5 us each:
// beside a prefix in tiles of 128 rows (128 questions of up to 512 keys behind 32768: 189 -> 162
// us; 64 of 1000 behind 8000: 80 -> 92), and in tiles of 64, which is shorter (75 of 4 behind
// 8705: 32.4 -> 28.3; 32 of 500 behind 4000: 37.9 -> 43.1).
constexpr int kBesideTiles = 16, kBesideTiles64 = 3;

// A wave's sequence and kv head, whole: its keys one tile after the other through the wave's
// part of a workgroup's LDS, as much as the prefix's tiles take.
template <typename T, int HD, int LDS>
struct Beside {
  static constexpr int MF = kBesideRows, KT = kPagedTokenTile;
  typedef WaveRows<T, HD, MF, KT, true> W;
  typedef Loader<T, HD, MF, KT> L;
  static constexpr int kTile = KT * Row<T, HD, MF>::kBytes, kWave = 2 * kTile;
  static constexpr int kWaves = LDS / kWave;

  static __device__ __forceinline__ void run(const PagedArgs &a, const AttnArgs &t, char *smem,
                                             int wave, int pair, const Pieces &out) {
    const int lane = threadIdx.x & 63, G = a.kv_heads, b = pair / G, g = pair % G;
    if (wave >= kWaves || b >= a.batch) return;
    const PagedSeq s = seq_of(a, b);
    const int two = two_of(t, b);
    const PagedRange rg = paged_range(s, t.window, two - t.prefix, KT);
    if (s.bad || s.n == 0) return;  // k_paged_merge sets such rows
    L load;
    load.begin(a);
    char *mine = smem + wave * kWave;
    const GroupRow me = group_row(t, lane % MF);
    const bool live = me.i < s.n;
    const int h = g * t.group + me.r, p0 = t.prefix + s.len - s.n;
    typename W::Query y;
    W::load(y, t, live ? t.q + (s.row0 + me.i) * t.ldq + (int64_t)h * a.hd : nullptr, a.hd, h);
    PageIds ids;
    auto issue = [&](int k) {
      const int j = rg.lo + k * KT;
      ids.cover(a, a.pages + b * a.cols, j, s.len, t.prefix);
      load.tile(a, ids, g * a.sh, j, s.len - 1, 0, 1, mine, mine + kTile);
    };
    issue(0);
    W r;
    r.begin(t, y, live ? p0 + me.i : -1, live ? two : 0, p0, p0 + s.n - 1, two, two);
    for (int k = 0; k < rg.n; k++) {
      wait_dma<0>();
      const int jp = t.prefix + rg.lo + k * KT;
      if (r.any(jp, t.window)) r.tile(t, mine, mine + kTile, jp, t.prefix + s.len);
      asm volatile("" ::: "memory");  // the stage is read before it is filled again
      if (k + 1 < rg.n) issue(k + 1);
    }
    const bool fine = r.end() && !ids.missed(a, t, r);
    if (live) {
      const int64_t slot = (int64_t)pair * MF + lane % MF;
      r.store(out.o + slot * a.hd, a.hd, 1.0f);
      if (lane < MF) put_ml(out, slot, r.m, fine ? r.l : __builtin_nanf(""));
    }
  }
};
template <typename T, int HD, int MF, int NG>
__global__ void __launch_bounds__(256 * NG, 2) k_paged_prefix(PagedArgs a, AttnArgs t,
                                                              PrefixPlan pl) {
  typedef Prompt<T, HD, MF, NG> P;
  typedef typename P::W W;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % 4;
  const int G = a.kv_heads, R = t.group;
  if ((int)blockIdx.x < pl.beside) {
    typedef Beside<T, HD, P::kLds> B;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    B::run(a, t, smem, w, blockIdx.x * min(4 * NG, B::kWaves) + w, pl.own);
    return;
  }
  const int id = blockIdx.x - pl.beside, z = id / pl.blocks, place = id % pl.blocks;
  const int g = place % G, tile = place / G;  // a head's workgroups share an XCD
  typename P::L load;
  load.begin(a);
  const int k = tile * P::kRows + wave * W::kRows + lane % W::kRows;
  const bool live = k < a.tokens * R;
  const int row = k / R, h = g * R + k % R;
  typename W::Query y;
  W::load(y, t, live ? t.q + row * t.ldq + (int64_t)h * a.hd : nullptr, a.hd, h);
  W r;
  begin_prefix(r, a, t, y, live, row);
  const int n = (t.prefix - t.seen + P::KT - 1) / P::KT;
  const int each = (n + pl.splits - 1) / pl.splits;
  if (!P::run(a, t, r, load, smem, nullptr, g * a.sh, {t.seen, n, 0, 0, 0},
              min(n, z * each),
              min(n, z * each + each)))
    return;
  const bool fine = r.end();
  if (live) {
    const int64_t slot = ((int64_t)z * a.tokens + row) * t.heads + h;
    r.store(pl.out.o + slot * a.hd, a.hd, 1.0f);
    if (lane < W::kRows) put_ml(pl.out, slot, r.m, fine ? r.l : __builtin_nanf(""));
  }
}

// Tile number p of the batch's: those that end at a later key first, which are the long ones
// where nothing limits what a row sees.  (-1 behind the last.)  A batch of more than 64, or
// `sorted` false: in the sequences' order.  Two prompts of 1024 rows 52.7 us, in the sequences'
// order 63.6; where every workgroup has a CU the order does not matter and is not looked for.
template <int KT, int ROWS>
__device__ __forceinline__ int tile_of_place(Seqs &q, const PagedArgs &a, const AttnArgs &t,
                                             bool sorted, int p, int *tile) {
  if (!sorted || a.batch > 64) {
    int before;
    const int b = q.template find<KT>(
        a, t, [&](const PagedSeq &s, const PagedRange &) {
          return paged_tiles_of(s, t.group, ROWS);
        }, p, &before);
    *tile = p - before;
    return b;
  }
  q.template look<KT>(a, t, 0);
  auto behind = [&](int x) { return paged_tiles_behind(q.s, t.group, ROWS, x); };
  int lo = -1, hi = a.max_kv;  // more than p tiles end behind lo, p or fewer behind hi
  if (__builtin_amdgcn_readlane(wave_scan(behind(lo)), 63) <= p) return -1;
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (__builtin_amdgcn_readlane(wave_scan(behind(mid)), 63) > p) lo = mid;
    else hi = mid;
  }
  const int later = behind(hi), here = behind(lo) - later;
  const int r = p - __builtin_amdgcn_readlane(wave_scan(later), 63), upto = wave_scan(here);
  const int b = __builtin_ctzll(__ballot(upto > r));
  *tile = __builtin_amdgcn_readlane(paged_tiles_of(q.s, t.group, ROWS) - later + upto - here, b) -
          1 - r;
  return b;
}

// splits: parts of the keys; with more than one, pieces [splits][tokens][heads].
struct PromptPlan {
  int splits;
  int mirror;     // workgroups of a round: the second round begins with the shortest, so that the
                  // two that share a CU are a long and a short one (0: none; the uneven prompts
                  // 153.9 -> 140.1 us, 1024 rows of 4 heads on 8 37.8 -> 38.6)
  bool sorted;
  Pieces out;
};

template <typename T, int HD, int MF, int NG>
__global__ void __launch_bounds__(256 * NG, 2) k_paged_prompt(PagedArgs a, AttnArgs t,
                                                              PromptPlan pl) {
  typedef Prompt<T, HD, MF, NG> P;
  typedef typename P::W W;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % 4;
  const int G = a.kv_heads, R = t.group;
  const int m = pl.mirror, bid = blockIdx.x;
  const int id = bid >= m && bid < 2 * m ? 3 * m - 1 - bid : bid;
  const int g = id % G, place = id / G;
  Seqs seqs;
  int tile;
  const int b = tile_of_place<P::KT, P::kRows>(seqs, a, t, pl.sorted, place, &tile);
  if (b < 0) return;
  const PagedSeq s = seqs.seq(b);
  const int two = seqs.two_way(b), z = blockIdx.y;
  if (s.bad) {  // (k_paged_merge does so itself)
    if (pl.splits == 1 && threadIdx.x < 64) refuse_rows(a, t, s, g);
    return;
  }
  typename P::L load;
  load.begin(a);
  const int first = tile * P::kRows, rows = s.n * R;
  const PagedKeys keys = paged_keys(s, t.prefix, R, t.window, two, first, P::kRows, P::KT);
  const int all = keys.na + keys.nb, each = (all + pl.splits - 1) / pl.splits;
  const int f = first + wave * W::kRows, k = f + lane % W::kRows;
  const bool live = k < rows, some = f < rows;
  const int i = k / R, h = g * R + k % R;
  typename W::Query y;
  W::load(y, t, live ? t.q + (s.row0 + i) * t.ldq + (int64_t)h * a.hd : nullptr, a.hd, h);
  const int p = t.prefix + s.len - s.n;
  W r;
  r.begin(t, y, live ? p + i : -1, live ? two : 0, some ? p + f / R : INT32_MAX,
          some ? p + min(f + W::kRows - 1, rows - 1) / R : -1, some ? two : INT32_MAX,
          some ? two : 0);
  if (!P::run(a, t, r, load, smem, a.pages + b * a.cols, g * a.sh, keys, min(all, z * each),
              min(all, z * each + each)))
    return;
  const bool fine = r.end();
  if (pl.splits == 1) {
    if (live && fine)
      r.store(t.out + (s.row0 + i) * t.ldo + (int64_t)h * a.hd, a.hd, inverse(r.l));
    uint64_t again = __ballot(live && !fine && lane < W::kRows);
    while (again) {
      const int u = f + __builtin_ctzll(again);
      again &= again - 1;
      redo_row<T>(a, t, b, s, u / R, g * R + u % R);
    }
  } else if (live) {
    const int64_t slot = ((int64_t)z * a.tokens + s.row0 + i) * t.heads + h;
    r.store(pl.out.o + slot * a.hd, a.hd, 1.0f);
    if (lane < W::kRows) put_ml(pl.out, slot, r.m, fine ? r.l : __builtin_nanf(""));
  }
}

// ---------------------------------------------------------------------------
// Rows from their pieces, in the pieces' order, a wave per row and head.  Bound by latency: 5 us
// after a token of one sequence, 7 for 4096 rows of 20 pieces; the sums are loaded along with
// the statistics that weigh them (30.7 -> 25.8 us for a token of 60000 keys with all launches).
// ---------------------------------------------------------------------------
struct MergePlan {
  TokenPlan token;    // token.waves: 0 without them
  int mf;
  int splits;         // of the other kernels' pieces; 0 without them
  Pieces split;
  bool beside;        // the prefix kernel has the sequences' own keys, pieces in token.out
};

// NW waves a row and head, each with every NW-th piece.  hd values of a piece take 32 lanes (16
// for up to 64 of them), so that a wave reads two (four) at a time.
template <typename T, int NW>
__global__ void __launch_bounds__(256) k_paged_merge(PagedArgs a, AttnArgs t, MergePlan pl) {
  constexpr int KT = kPagedTokenTile;
  __shared__ __attribute__((aligned(16))) float sm[4][kPagedMergeRow];
  // in one round of loads (left to itself the compiler takes four, some after the row's sequence
  // is known: 5.2 us after a token of one sequence, 5.0 so)
  kernarg_fence(a.k, a.v, a.sp, a.sh, a.sr, a.num_pages, a.shift, a.start, a.kv_len, a.pages,
                a.cols, a.batch, a.tokens, a.max_q, a.max_kv, a.kv_heads, a.hd);
  kernarg_fence(t.out, t.ldo, t.heads, t.group, t.ppages, t.prefix, t.window, t.two);
  kernarg_fence(pl.token.waves, (int)pl.token.keep, pl.token.flat, pl.token.sets, pl.token.out.o,
                pl.token.out.ml, pl.mf, pl.splits, pl.split.o, pl.split.ml, (int)pl.beside);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % NW;
  const uint32_t rh = blockIdx.x * (4 / NW) + wave / NW;
  const int row = rh / (uint32_t)t.heads, h = rh % (uint32_t)t.heads, lane = threadIdx.x & 63;
  if (row >= a.tokens) return;
  const int G = a.kv_heads, g = h / t.group;
  Seqs seqs;
  int b;
  if (a.batch < 64) {
    const int first = lane <= a.batch ? a.start[lane] : INT32_MAX;
    seqs.look<KT>(a, t, 0);
    b = __popcll(__ballot(first <= row)) - 1;
    if (b < 0 || b >= a.batch) return;
  } else {
    b = min(max(0, seq_of_row_wave(a, row)), a.batch - 1);
  }
  auto share = [&](const PagedSeq &, const PagedRange &r) { return r.n * G; };
  int before = 0, total = 0;
  if (pl.token.waves) total = seqs.length<KT>(a, t, share, b, &before);
  seqs.look<KT>(a, t, b);
  const PagedSeq s = seqs.seq(b);
  auto merge = [&](int i) {  // whether the row's sums are not finite
    float *out = t.out + row * t.ldo + (int64_t)h * a.hd;
    if (s.bad) {
      if (part == 0 && lane < a.hd) out[lane] = __builtin_nanf("");
      if (part == 0 && lane + 64 < a.hd) out[lane + 64] = __builtin_nanf("");
      return false;
    }
    // pieces of the prefix, the token kernel's or the prefix kernel's, then of its own keys
    int lead = pl.splits, n = lead, w0 = 0, wp = 0;
    const int flat = pl.token.flat, pairs = pl.token.sets * G;
    const int c = i * t.group + h % t.group, f0 = s.row0 * t.group + c;
    const int set = flat ? g * pl.token.sets + f0 / pl.mf : 0;
    if (pl.token.waves) {
      const uint32_t each = paged_each(total + flat * pairs, pl.token.waves);
      const int tiles = seqs.range(b).n, x0 = flat * pairs + before + g * tiles;
      if (flat) {
        wp = set * flat / each;
        lead = (set * flat + flat - 1) / each - wp + 1;
      }
      w0 = x0 / each;
      const int w1 = (x0 + tiles - 1) / each;
      if (w0 == w1 && !pl.token.keep) return false;  // stored by its wave
      n = lead + w1 - w0 + 1;
    }
    n += pl.beside;
    auto place = [&](int k) -> int64_t {
      if (k >= lead && pl.beside) return ((int64_t)b * G + g) * kBesideRows + c;
      if (k < lead && flat) return token_slot(true, wp + k, set, false) * pl.mf + f0 % pl.mf;
      if (k < lead) return ((int64_t)k * a.tokens + row) * t.heads + h;
      const int u = k - lead;
      return token_slot(pl.token.keep, w0 + u, pairs + (int64_t)b * G + g, u == 0) * pl.mf + c;
    };
    const int lpp = a.hd > 64 ? 32 : 16, np = 64 / lpp, d = 4 * (lane % lpp), sub = lane / lpp;
    float m = kNegInf, l = 0.0f;
    f4 o = {0, 0, 0, 0};
    for (int base = part; base < n; base += 64 * NW) {
      const int k = base + lane * NW, cnt = min(64, (n - base + NW - 1) / NW);
      float pm = kNegInf, f = 0.0f;
      int64_t at = 0;
      const float *src = nullptr;
      if (lane < cnt) {
        const Pieces &p = k < lead && !flat ? pl.split : pl.token.out;
        at = place(k);
        pm = p.ml[2 * at];
        f = p.ml[2 * at + 1];
        src = p.o + at * a.hd;
      }
      f4 v[8];
      auto read = [&](int q) {
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const int from = min(q + u * np + sub, cnt - 1);
          const float *po = (const float *)__shfl((unsigned long long)src, from);
          v[u] = *(const f4 *)(po + (d < a.hd ? d : 0));
        }
      };
      read(0);  // in flight with m and l
      float top = pm;
#pragma unroll
      for (int w = 1; w < 64; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
      const float next = fmaxf(m, top), ref = next == kNegInf ? 0.0f : next;
      const float old = __builtin_amdgcn_exp2f(m - ref), wt = __builtin_amdgcn_exp2f(pm - ref);
      float sum = lane < cnt ? f * wt : 0.0f;
#pragma unroll
      for (int w = 1; w < 64; w *= 2) sum += __shfl_xor(sum, w);
      m = next;
      l = l * old + sum;
      o *= old;
      for (int q = 0;;) {
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const int want = q + u * np + sub;
          const float g = __shfl(wt, min(want, cnt - 1)), pw = want < cnt ? g : 0.0f;
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] = fmaf(pw, v[u][e], o[e]);
        }
        q += 8 * np;
        if (q >= cnt) break;
        read(q);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (lpp == 16) o[e] += __shfl_xor(o[e], 16);
      o[e] += __shfl_xor(o[e], 32);
    }
    if constexpr (NW > 1) {
      if (lane < lpp && d < a.hd) *(f4 *)&sm[wave][d] = o;
      if (lane == 0) sm[wave][a.hd] = m, sm[wave][a.hd + 1] = l;
      __syncthreads();
      if (part) return false;
      float top = kNegInf;
#pragma unroll
      for (int w = 0; w < NW; w++) top = fmaxf(top, sm[w][a.hd]);
      const float ref = top == kNegInf ? 0.0f : top;
      l = 0.0f;
      o = f4{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const float f = __builtin_amdgcn_exp2f(sm[w][a.hd] - ref);
        l = fmaf(sm[w][a.hd + 1], f, l);
        if (d < a.hd)
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] = fmaf(sm[w][d + e], f, o[e]);
      }
    }
    bool fine = paged_finite(l);
#pragma unroll
    for (int e = 0; e < 4; e++) fine = fine && paged_finite(o[e]);
    if (!__all(fine)) return true;
    const float f = inverse(l);
    if (lane < lpp && d < a.hd) *(f4a4 *)(out + d) = f4a4{o[0] * f, o[1] * f, o[2] * f, o[3] * f};
    return false;
  };
  // (not in: another sequence's row, or none's)
  const bool again = paged_in(s, row) ? merge(row - s.row0) : part == 0;
  if (again) row_anew<T>(a, t, row, h);
}

// ---------------------------------------------------------------------------
// Attention, a wave per row and head: caches whose rows lie too far apart for a tile's loads.
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) k_paged_rows(PagedArgs a, AttnArgs t) {
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = (int)(r / t.heads), h = (int)(r % t.heads);
  if (row >= a.tokens) return;
  row_anew<T>(a, t, row, h);
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
template <typename P, typename K, typename Plan>
int launch_prompt(mmnb_ctx *ctx, K kern, const PagedArgs &a, const AttnArgs &t, const Plan &pl,
                  int64_t blocks, int64_t parts) {
  if (int rc = allow_lds(kern, P::kLds)) return rc;
  return launch(ctx, kKernPagedAttn, kern, dim3((unsigned)blocks, (unsigned)parts),
                dim3(P::kThreads), P::kLds, a, t, pl);
}

// Device memory for `rows` pieces.
inline int pieces_get(mmnb_ctx *ctx, int64_t rows, int hd, Pieces *p) {
  void *buf = nullptr;
  const size_t need = (size_t)rows * (hd + 2) * 4;
  if (int rc = scratch_get(ctx, kPagedScratch, std::max(need, kPagedScratchBytes), &buf))
    return rc;
  p->o = (float *)buf;
  p->ml = p->o + rows * hd;
  return MMNB_OK;
}

// Four waves a row where one would take more than two rounds of loads (two sequences of up to
// 131071 keys, 64 pieces a row: 67.5 us with one wave, 7.5 with four).
template <typename T>
int launch_merge(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t, const MergePlan &mp,
                 int64_t pieces) {
  const int64_t all = (int64_t)a.tokens * t.heads;
  if (pieces > 32)
    return launch(ctx, kKernPagedMerge, k_paged_merge<T, 4>, dim3((unsigned)all), dim3(256), 0, a,
                  t, mp);
  return launch(ctx, kKernPagedMerge, k_paged_merge<T, 1>, dim3((unsigned)((all + 3) / 4)),
                dim3(256), 0, a, t, mp);
}

// Sets the parts that the prefix is cut into; the tiles of keys that all workgroups have.
template <typename P>
int64_t prefix_plan(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t, int *splits) {
  const int64_t rows = (int64_t)a.tokens * t.group;
  const int64_t blocks = a.kv_heads * ((rows + P::kRows - 1) / P::kRows);
  const int64_t tiles = (t.prefix - t.seen + P::KT - 1) / P::KT;
  *splits = (int)paged_splits(blocks, tiles, P::kThreads / 256, ctx->cu_count * P::kPerCu);
  return blocks * tiles;
}
template <typename T, int HD, typename P, typename K>
int launch_prefix(mmnb_ctx *ctx, K kern, const PagedArgs &a, const AttnArgs &t,
                  const MergePlan &mp) {
  const int64_t rows = (int64_t)a.tokens * t.group;
  const int64_t blocks = a.kv_heads * ((rows + P::kRows - 1) / P::kRows);
  constexpr int waves = std::min(P::kThreads / 64, Beside<T, HD, P::kLds>::kWaves);
  PrefixPlan pl = {};
  pl.splits = mp.splits;
  pl.blocks = (int)blocks;
  pl.beside = mp.beside ? (int)(((int64_t)a.batch * a.kv_heads + waves - 1) / waves) : 0;
  pl.out = mp.split;
  pl.own = mp.token.out;
  return launch_prompt<P>(ctx, kern, a, t, pl, pl.beside + blocks * mp.splits, 1);
}

// Few rows of each sequence.
template <typename T, int HD>
int attention_token(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t) {
  typedef TokenShape<T, HD> S;
  const int64_t all = (int64_t)a.tokens * t.heads, pairs = (int64_t)a.batch * a.kv_heads;
  const int64_t rows = (int64_t)a.tokens * t.group, each = (int64_t)a.max_q * t.group;
  MergePlan mp = {};
  TokenPlan &tp = mp.token;
  tp.waves = ctx->cu_count * S::kPerCu * S::kWaves;
  tp.keep = t.prefix > 0;
  // A few tiles after each other cost less than merging what waves made of them: 60 keys of 8
  // sequences on 8 heads 13.4 -> 9.9 us whole, 160 keys 12.2 -> 11.8, 300 keys 13.6 -> 19.3; and
  // more where pairs of sequence and head are as many as half the waves: 160 keys of 64
  // sequences 21.0 -> 13.4, 500 keys 33.0 -> 28.7.
  const int64_t tiles = (a.max_kv + kPagedTokenTile - 1) / kPagedTokenTile;
  tp.whole = !t.prefix && (tiles <= 5 || (tiles <= 16 && 2 * pairs >= tp.waves));
  // A prefix that is little work for all waves, though each set of MF rows reads it again, is a
  // sequence among the others: 33 talks behind 4001 keys (four tiles a wave) 27.5 us so, 33.2
  // with a launch of its own; 32 behind 4000 keys on 8 heads of 128 (eight) 41.7 and 35.4.
  mp.mf = each <= 16 ? 16 : 32;
  const int64_t sets = (rows + mp.mf - 1) / mp.mf;
  const int64_t flat = (t.prefix - t.seen + kPagedTokenTile - 1) / kPagedTokenTile;
  if (t.prefix && flat * sets * a.kv_heads <= 5 * tp.waves) {
    tp.flat = (int)flat;
    tp.sets = (int)sets;
  }
  const int64_t lead = (int64_t)tp.sets * a.kv_heads;
  bool wide = false;
  if (t.prefix && !tp.flat) {
    // Tiles of 128 rows read the prefix less often and are worth it where each CU has many:
    // 512 rows behind 32768 keys 192.0 us, in tiles of 64 196.4; 264 behind 4001 35.3 and 32.2.
    wide = rows > 192 &&
           prefix_plan<Prompt<T, HD, 32, 1>>(ctx, a, t, &mp.splits) >= 16 * ctx->cu_count;
    if (!wide) prefix_plan<Prompt<T, HD, 16, 2>>(ctx, a, t, &mp.splits);
    mp.beside = each <= kBesideRows && tiles <= (wide ? kBesideTiles : kBesideTiles64);
    if (mp.beside) tp.waves = 0;
  }
  const int64_t slots = mp.beside ? pairs * kBesideRows
                        : mp.mf * (tp.keep ? tp.waves + pairs + lead : 2 * (int64_t)tp.waves);
  if (int rc = pieces_get(ctx, slots + mp.splits * all, a.hd, &tp.out)) return rc;
  mp.split = {tp.out.o + slots * a.hd, tp.out.ml + slots * 2};
  if (mp.splits)
    if (int rc = wide ? launch_prefix<T, HD, Prompt<T, HD, 32, 1>>(
                            ctx, k_paged_prefix<T, HD, 32, 1>, a, t, mp)
                      : launch_prefix<T, HD, Prompt<T, HD, 16, 2>>(
                            ctx, k_paged_prefix<T, HD, 16, 2>, a, t, mp))
      return rc;
  if (mp.beside) return launch_merge<T>(ctx, a, t, mp, mp.splits + 1);
  if (int rc = mp.mf == 16 ? launch_token<T, HD, 16>(ctx, a, t, tp)
                           : launch_token<T, HD, 32>(ctx, a, t, tp))
    return rc;
  if (tp.whole) return MMNB_OK;
  // the pieces that a row has, if sequences are alike
  const int64_t run = (tp.flat * lead + tiles * pairs + tp.waves - 1) / tp.waves;
  return launch_merge<T>(ctx, a, t, mp, mp.splits + tp.flat / run + tiles / run + 1);
}

// Many rows.  Keys are cut where the parts' time and their merge are less than the whole's: 64
// rows of 4 heads on 8 over 4000 keys 73 us in one part, 23 in eight; 512 rows of their own 512
// keys 18.5 us in one, 41 in two, with the pieces' way through memory.
template <typename T, int HD, int MF, int NG>
int attention_prompt(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t) {
  typedef Prompt<T, HD, MF, NG> P;
  const int64_t blocks =
      a.kv_heads * paged_row_tiles(a.batch, a.tokens, a.max_q, t.group, P::kRows);
  PromptPlan pl = {};
  pl.splits = (int)paged_prompt_parts(blocks, ((int64_t)t.prefix + a.max_kv) / P::KT + 1, NG,
                                      (int64_t)a.tokens * t.heads * (a.hd + 2) * 4,
                                      ctx->cu_count * P::kPerCu);
  pl.sorted = blocks * pl.splits > ctx->cu_count;
  pl.mirror = blocks >= 2 * ctx->cu_count && blocks < 4 * ctx->cu_count ? ctx->cu_count : 0;
  if (pl.splits > 1)
    if (int rc = pieces_get(ctx, pl.splits * (int64_t)a.tokens * t.heads, a.hd, &pl.out))
      return rc;
  if (int rc = launch_prompt<P>(ctx, k_paged_prompt<T, HD, MF, NG>, a, t, pl, blocks, pl.splits))
    return rc;
  if (pl.splits == 1) return MMNB_OK;
  MergePlan mp = {};
  mp.splits = pl.splits;
  mp.split = pl.out;
  return launch_merge<T>(ctx, a, t, mp, mp.splits);
}

template <typename T, int HD>
int launch_attention(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t) {
  const int64_t most = (a.max_kv / kPagedTokenTile + 1) * (int64_t)a.batch * a.kv_heads;
  if ((int64_t)a.max_q * t.group <= kPagedTokenRows && most <= INT32_MAX / 2)
    return attention_token<T, HD>(ctx, a, t);
  auto blocks = [&](int rows) {
    return a.kv_heads * paged_row_tiles(a.batch, a.tokens, a.max_q, t.group, rows);
  };
  // 128 rows a workgroup from one and a half a CU on (424 of them, the window prompt: 334 us, in
  // 64 rows 406; 256 of them, 1024 rows over 4000 keys: 139 and 127).  64 rows on eight waves
  // where that leaves a CU to each (512 rows of 1000 keys on bf16: 31 us, on four 39; 1024 rows
  // of 1024 keys, two a CU: 46 and 36) and there is more than a tile for both halves (64 rows of
  // 64 keys: 10.4 and 9.3).
  if (2 * blocks(128) >= 3 * ctx->cu_count) return attention_prompt<T, HD, 32, 1>(ctx, a, t);
  return blocks(64) > ctx->cu_count || t.prefix + a.max_kv <= 128
             ? attention_prompt<T, HD, 16, 1>(ctx, a, t)
             : attention_prompt<T, HD, 16, 2>(ctx, a, t);
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
