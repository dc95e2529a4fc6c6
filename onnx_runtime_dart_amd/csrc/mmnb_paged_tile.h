// Attention of a wave's MF query rows over tiles of KT keys staged in LDS, on the matrix cores.
//
// Scores are computed transposed, S^T = K Q^T, so that a lane holds scores of one query alone
// (query lane % MF; its keys are those of lane group lane / MF): the running maximum is per
// lane, and rescaling the sums O^T = V^T P^T, whose columns are queries too, needs no exchange
// between lanes.  The scores' registers are P^T's operand as they stand: a product's result
// gives a lane four consecutive keys at a time, and the sum over keys may take them in any
// order as long as V^T's operand is read in the same one.
#pragma once

#include "mmnb_device.h"
#include "mmnb_paged.h"

namespace mmnb {

typedef short s4vec __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

__device__ __forceinline__ uint32_t lds_addr(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)p;
}
// Four rows of 16 two-byte values in LDS, transposed: lane i of each 16 points at values
// 4 (i % 4) .. of row i / 4 and gets column i's four rows.
__device__ __forceinline__ s4vec lds_tr4(const char *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4vec *)p);
}
// N addresses, each at two offsets, without the builtin, before which the compiler waits for
// every LDS DMA in flight, the next tile's too.
template <int O0, int O1, int N>
__device__ __forceinline__ void lds_tr(const uint32_t (&at)[N], s4vec (&lo)[N], s4vec (&hi)[N]) {
  static_assert(N >= 2 && N <= 4, "");
  if constexpr (N == 2)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
        "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1])
        : "v"(at[0]), "v"(at[1]), "n"(O0), "n"(O1)
        : "memory");
  else if constexpr (N == 3)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %6 offset:%9\n\tds_read_b64_tr_b16 %1, %6 offset:%10\n\t"
        "ds_read_b64_tr_b16 %2, %7 offset:%9\n\tds_read_b64_tr_b16 %3, %7 offset:%10\n\t"
        "ds_read_b64_tr_b16 %4, %8 offset:%9\n\tds_read_b64_tr_b16 %5, %8 offset:%10\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "n"(O0), "n"(O1)
        : "memory");
  else
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
        "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]),
          "=&v"(lo[3]), "=&v"(hi[3])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(O0), "n"(O1)
        : "memory");
}

// ---- operands
// A matrix operand of eight (four for binary32) consecutive values of the contraction, and how
// a binary32 value is held in it: fp16 as two terms (22 bits), bf16 as three (24 bits), each
// rounded to nearest.  K and V are exact in their own type, so that all products are exact and
// sums are binary32: results as near the definition as binary32 arithmetic gives, at two and
// three times the products.
template <typename T>
struct Operand;
template <>
struct Operand<float> {
  typedef f4 frag;
  static constexpr int kVals = 4, kTerms = 1;
  static __device__ __forceinline__ void split(const float (&x)[4], frag (&t)[1]) {
    t[0] = f4{x[0], x[1], x[2], x[3]};
  }
};
template <>
struct Operand<_Float16> {
  typedef half8 frag;
  static constexpr int kVals = 8, kTerms = 2;
  static __device__ __forceinline__ void split(const float (&x)[8], frag (&t)[2]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const _Float16 a = (_Float16)x[i];
      t[0][i] = a;
      t[1][i] = (_Float16)(x[i] - (float)a);
    }
  }
};
template <>
struct Operand<__bf16> {
  typedef bf8 frag;
  static constexpr int kVals = 8, kTerms = 3;
  static __device__ __forceinline__ void split(const float (&x)[8], frag (&t)[3]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const __bf16 a = (__bf16)x[i];
      const float r = x[i] - (float)a;
      const __bf16 b = (__bf16)r;
      t[0][i] = a;
      t[1][i] = b;
      t[2][i] = (__bf16)(r - (float)b);
    }
  }
};

template <int MF>
struct Acc;
template <>
struct Acc<32> {
  typedef f16v v;
};
template <>
struct Acc<16> {
  typedef f4 v;
};

template <int MF, typename V>
__device__ __forceinline__ void mfma(const half8 &a, const half8 &b, V &c) {
  if constexpr (MF == 32) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  else c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
template <int MF, typename V>
__device__ __forceinline__ void mfma(const bf8 &a, const bf8 &b, V &c) {
  if constexpr (MF == 32) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  else c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <int MF, typename V>
__device__ __forceinline__ void mfma(float a, float b, V &c) {
  if constexpr (MF == 32) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  else c = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
template <int MF, typename V>
__device__ __forceinline__ void mfma(const f4 &a, const f4 &b, V &c) {
#pragma unroll
  for (int i = 0; i < 4; i++) mfma<MF>(a[i], b[i], c);
}

// ---- tiles in LDS
// A key's (value's) row is kChunks pieces of 16 bytes, of which the first hd values are
// loaded; piece c lies at c ^ swz(row), so that what the operand reads touch at once, 256 bytes,
// lies in different banks: for keys a piece of 16 rows, for values 64 (MF = 16: 32) bytes of
// four (eight) rows, or binary32 words of two (four) rows four apart.  (With keys at c ^ row % 8
// and values 32 bytes apart half the LDS's cycles were conflicts; now none is.)  A DMA
// instruction fills kRows rows.
template <typename T, int HD, int MF>
struct Row {
  static constexpr int kVals = 16 / (int)sizeof(T);
  static constexpr int kUsed = HD / kVals;
  static constexpr int kChunks = kUsed <= 8 ? 8 : kUsed <= 16 ? 16 : 32;
  static constexpr int kBytes = kChunks * 16;
  static constexpr int kRows = 64 / kChunks;
  static __device__ __forceinline__ int swz_k(int row) {
    return kChunks == 8 ? (row >> 1) & 7 : row & 15;
  }
  static __device__ __forceinline__ int swz_v(int row) {
    if (sizeof(T) == 4) return MF == 32 ? ((row >> 2) & 1) << 3 : ((row >> 2) & 3) << 2;
    if (kChunks == 8) return MF == 32 ? ((row >> 1) & 1) << 2 : ((row >> 1) & 3) << 1;
    return MF == 32 ? (row & 3) << 2 : (row & 7) << 1;
  }
};

// The pages of a sequence (or of the prefix) as a wave reads them: 64 numbers at a time, one
// per lane.
struct PageIds {
  const int32_t *table = nullptr;
  int base = 0, ids = 0, lost = -1;
  // Numbers of the pages from that of key j on (j a multiple of a tile); keys from `end` on are
  // not looked up.  Key 0 has position `off`.
  __device__ __forceinline__ void cover(const PagedArgs &a, const int32_t *t, int j, int end,
                                        int off) {
    const int first = (j >> a.shift) & ~63;
    if (t == table && first == base) return;
    table = t;
    base = first;
    const int i = first + (threadIdx.x & 63);
    bool out = false;
    ids = (int64_t)i << a.shift < end ? paged_page(t[i], a.num_pages, &out) : 0;
    lost = paged_lose(lost, out, i, a.shift, off);
  }
  // Whether the wave's rows miss a key.
  template <typename W>
  __device__ __forceinline__ bool missed(const PagedArgs &a, const AttnArgs &t, const W &r) const {
    return __any(paged_missed(lost, a.shift, r.pmin, t.window, r.tmax));
  }
  __device__ __forceinline__ int of(const PagedArgs &a, int j) const {
    return __builtin_amdgcn_readlane(ids, (j >> a.shift) - base);
  }
};

// Keys [j0, j0 + KT) of one head, and their values, into LDS at kd and vd, by wave w of nw, each
// of which takes its part of the DMA instructions.  Rows past `last` repeat it, so that what
// lies behind a sequence in its last page never enters a product; pieces past hd repeat the
// last one, whose products meet zeros of the query, or are not stored.
template <typename T, int HD, int MF, int KT>
struct Loader {
  typedef Row<T, HD, MF> R;
  static constexpr int kIns = KT / R::kRows;  // DMA instructions for K, and for V
  int lr, top;      // the lane's row of an instruction; the last piece of a row
  int xk, xv;       // ... its piece in the first instruction's rows
  uint32_t row;     // bytes of a row

  __device__ __forceinline__ void begin(const PagedArgs &a) {
    const int lane = threadIdx.x & 63, c = lane % R::kChunks;
    lr = lane / R::kChunks;
    xk = c ^ R::swz_k(lr);
    xv = c ^ R::swz_v(lr);
    top = a.hd / R::kVals - 1;
    row = (uint32_t)a.sr * (uint32_t)sizeof(T);
  }
  // A lane's bytes from the begin of its row of instruction u (the swizzles of an instruction's
  // first row and of lr have no bits in common).
  __device__ __forceinline__ uint32_t at_k(int u) const {
    return min(xk ^ R::swz_k(u * R::kRows), top) * 16;
  }
  __device__ __forceinline__ uint32_t at_v(int u) const {
    return min(xv ^ R::swz_v(u * R::kRows), top) * 16;
  }
  __device__ __forceinline__ void tile(const PagedArgs &a, const PageIds &ids, int64_t head,
                                       int j0, int last, int w, int nw, char *kd,
                                       char *vd) const {
    const int pg = 1 << a.shift;
    const int u0 = w * (kIns / nw);
    if (j0 + KT - 1 <= last && pg >= R::kRows) {
      const uint32_t lo = (uint32_t)lr * row, step = R::kRows * row;
      const int ins = pg >= KT ? kIns : pg / R::kRows;  // instructions of a page
      __amdgpu_buffer_rsrc_t kr, vr;
      uint32_t soff = 0;
      auto page = [&](int u) {
        const int jj = j0 + u * R::kRows;
        const int64_t at =
            (ids.of(a, jj) * a.sp + (int64_t)(jj & (pg - 1)) * a.sr + head) * (int)sizeof(T);
        kr = buf_rsrc(a.k + at);
        vr = buf_rsrc(a.v + at);
        soff = 0;
      };
      page(u0);
#pragma unroll
      for (int i = 0; i < kIns; i++) {
        if (i >= kIns / nw) break;
        const int u = u0 + i;
        if (i > 0 && ins < kIns && (u & (ins - 1)) == 0) page(u);
        dma16_buf(kr, lo + at_k(u), soff, kd + u * 1024);
        dma16_buf(vr, lo + at_v(u), soff, vd + u * 1024);
        soff += step;
      }
      return;
    }
    // rows of an instruction may lie in several pages, or past the last key
#pragma unroll 1
    for (int n = 0; n < kIns / nw; n++) {
      const int u = u0 + n, jj = j0 + u * R::kRows;
      for (int q = 0; q < R::kRows; q += pg) {
        const int jb = min(jj + q, last);
        const uint32_t r = max(0, min(lr - q, last - jj - q));
        const int64_t at =
            (ids.of(a, jb) * a.sp + (int64_t)(jb & (pg - 1)) * a.sr + head) * (int)sizeof(T);
        const uint32_t k = at_k(u), v = at_v(u);
        if (lr >= q && lr < q + pg) {
          dma16_buf(buf_rsrc(a.k + at), r * row + k, 0, kd + u * 1024);
          dma16_buf(buf_rsrc(a.v + at), r * row + v, 0, vd + u * 1024);
        }
      }
    }
  }
  // DMA instructions of a wave per tile (a tile at a sequence's end, or of pages below kRows
  // keys, takes as many or more)
  static constexpr int per_wave(int nw) { return 2 * kIns / nw; }
};

// Waits until at most N of the wave's DMA loads are in flight.
template <int N>
__device__ __forceinline__ void wait_dma() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// ---- a wave's rows
// DMA: whether the wave has LDS DMA of later tiles in flight that it may not wait for when it
// reads values (a wave by itself); else the reads of a step are in flight with the products of
// the one before.
template <typename T, int HD, int MF, int KT, bool DMA>
struct WaveRows {
  typedef Operand<T> Op;
  typedef Row<T, HD, MF> R;
  typedef typename Op::frag frag;
  typedef typename Acc<MF>::v acc;
  static constexpr int kRows = MF;
  static constexpr int kG = 64 / MF;              // lane groups along the contraction
  static constexpr int kC = MF * MF / 64;         // a product's registers
  static constexpr int kNS = HD / (Op::kVals * kG);  // steps of the product over the head
  static constexpr int kNB = KT / MF;             // blocks of keys
  static constexpr int kND = HD / MF;             // blocks of the head
  static constexpr int kVals = kND;               // operands of values in a step
  // Weights are exp2(z - ref) with ref = m - kLift: on fp16 operands they lie between 2^-24 and
  // 2^15, so that small ones keep their bits.  The maximum that they are relative to may lag
  // kLag behind the true one, which saves most rescalings of the sums (8192-token prompt with a
  // lag of 5 971 us, of 2 983, of 1 991).
  static constexpr float kLift = sizeof(T) == 4 ? 0.0f : Op::kTerms == 2 ? 10.0f : 0.0f;
  static constexpr float kLag = 5.0f;

  frag q[kNS][Op::kTerms];
  acc o[kND];
  float m, l, mulq, slope;
  int p, two;                        // the lane's row
  int pmin, pmax, tmin, tmax;        // over the wave's rows

  // Which keys a score register holds: key_of(blk, i) + 4 (lane / MF)
  static __device__ __forceinline__ int key_of(int blk, int i) {
    return MF == 32 ? blk * 32 + 8 * (i / 4) + i % 4 : blk * 16 + i;
  }

  // What the lane loads of its row; the loads may be in flight while others are issued.
  struct Query {
    float x[kNS][Op::kVals], slope;
  };
  // src: the lane's row of queries of head h (null: none).
  static __device__ __forceinline__ void load(Query &y, const AttnArgs &t, const float *src,
                                              int hd, int h) {
    const int kg = ((int)threadIdx.x & 63) / MF;
    const bool live = src != nullptr;
    const float *from = live ? src : t.q;  // all lanes load, so that no branch parts the loads
#pragma unroll
    for (int s = 0; s < kNS; s++) {
      const int d = (kG * s + kg) * Op::kVals;
      const bool in = live && d < hd;
#pragma unroll
      for (int i = 0; i < Op::kVals; i += 4) {
        const f4a4 v = *(const f4a4 *)(from + (in ? d + i : 0));
#pragma unroll
        for (int k = 0; k < 4; k++) y.x[s][i + k] = in ? v[k] : 0.0f;
      }
    }
    y.slope = live && t.slopes ? t.slopes[h] : 0.0f;
  }
  // The row's position and the keys that all see (-1 and 0 without a row), and the least and
  // greatest of these over the wave's rows.
  __device__ __forceinline__ void begin(const AttnArgs &t, Query &y, int pos, int two_way,
                                        int p0, int p1, int t0, int t1) {
    mulq = t.capped ? t.in_mul : t.mul;
    if constexpr (Op::kTerms == 1) {
      // Here the loads are waited for; at the first product, in a loop, the compiler would wait
      // for all that is in flight by then.
#pragma unroll
      for (int s = 0; s < kNS; s++)
#pragma unroll
        for (int i = 0; i < Op::kVals; i++) asm volatile("" : "+v"(y.x[s][i]));
    }
    if constexpr (Op::kTerms == 2) {
      // the row's largest value to 2^14, so that the terms of all that counts are normal
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < kNS; s++)
#pragma unroll
        for (int i = 0; i < Op::kVals; i++) top = fmaxf(top, fabsf(y.x[s][i]));
#pragma unroll
      for (int w = MF; w < 64; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
      const int e = top > 0.0f && top < __builtin_inff()
                        ? max(-112, min(100, 14 - __builtin_amdgcn_frexp_expf(top) + 1))
                        : 0;
#pragma unroll
      for (int s = 0; s < kNS; s++)
#pragma unroll
        for (int i = 0; i < Op::kVals; i++) y.x[s][i] = __builtin_amdgcn_ldexpf(y.x[s][i], e);
      mulq = __builtin_amdgcn_ldexpf(mulq, -e);
    }
#pragma unroll
    for (int s = 0; s < kNS; s++) Op::split(y.x[s], q[s]);
    slope = y.slope * kLog2e;
    p = pos;
    two = two_way;
    pmin = p0, pmax = p1, tmin = t0, tmax = t1;
    m = kNegInf;
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < kND; d++)
#pragma unroll
      for (int i = 0; i < kC; i++) o[d][i] = 0.0f;
  }
  // The same where the rows belong to any sequences.
  __device__ __forceinline__ void begin_any(const AttnArgs &t, Query &y, bool live, int pos,
                                            int two_way) {
    int p0 = live ? pos : INT32_MAX, p1 = live ? pos : -1;
    int t0 = live ? two_way : INT32_MAX, t1 = live ? two_way : 0;
#pragma unroll
    for (int w = 1; w < MF; w *= 2) {
      p0 = min(p0, __shfl_xor(p0, w));
      p1 = max(p1, __shfl_xor(p1, w));
      t0 = min(t0, __shfl_xor(t0, w));
      t1 = max(t1, __shfl_xor(t1, w));
    }
    begin(t, y, live ? pos : -1, live ? two_way : 0, __builtin_amdgcn_readfirstlane(p0),
          __builtin_amdgcn_readfirstlane(p1), __builtin_amdgcn_readfirstlane(t0),
          __builtin_amdgcn_readfirstlane(t1));
  }

  // Whether any row sees a key at positions [j, j + KT), and whether all rows see all of them.
  __device__ __forceinline__ bool any(int j, int window) const {
    return (j <= pmax && (window == 0 || pmin - (j + KT - 1) < window)) || j < tmax;
  }
  __device__ __forceinline__ bool all(int j, int window) const {
    return (j + KT - 1 <= pmin && (window == 0 || pmax - j < window)) || j + KT <= tmin;
  }

  // One tile: keys at positions jp .. of which those from `end` on are no keys.
  __device__ __forceinline__ void tile(const AttnArgs &t, const char *kd, const char *vd, int jp,
                                       int end) {
    const int lane = threadIdx.x & 63, c = lane % MF, kg = lane / MF;
    acc s[kNB];
#pragma unroll
    for (int b = 0; b < kNB; b++)
#pragma unroll
      for (int i = 0; i < kC; i++) s[b][i] = 0.0f;
    {
      const char *row = kd + c * R::kBytes;
      const int x = (kg ^ R::swz_k(c)) << 4;
      frag k[2][kNB];
      auto read = [&](int st) {
        const char *at = row + (x ^ ((kG * st) << 4));
#pragma unroll
        for (int b = 0; b < kNB; b++) k[st & 1][b] = *(const frag *)(at + b * MF * R::kBytes);
      };
      read(0);
#pragma unroll
      for (int st = 0; st < kNS; st++) {
        if (st + 1 < kNS) read(st + 1);
        __builtin_amdgcn_sched_barrier(0);  // ahead of the products that hide it
#pragma unroll
        for (int w = 0; w < Op::kTerms; w++)
#pragma unroll
          for (int b = 0; b < kNB; b++) mfma<MF>(k[st & 1][b], q[st][w], s[b]);
      }
    }
    float mul = mulq;
    const int j1 = jp + 4 * kg;
    if (t.capped) {
#pragma unroll
      for (int b = 0; b < kNB; b++)
#pragma unroll
        for (int i = 0; i < kC; i++) s[b][i] = t.mul * paged_tanh(s[b][i] * mulq);
      mul = 1.0f;
    }
    if (t.slopes) {
#pragma unroll
      for (int b = 0; b < kNB; b++)
#pragma unroll
        for (int i = 0; i < kC; i++) {
          const int far = p - (j1 + key_of(b, i));
          s[b][i] = mul * s[b][i] - slope * (float)(far < 0 ? -far : far);
        }
      mul = 1.0f;
    }
    if (jp + KT > end || !all(jp, t.window)) {
#pragma unroll
      for (int b = 0; b < kNB; b++)
#pragma unroll
        for (int i = 0; i < kC; i++) {
          const int j = j1 + key_of(b, i);
          s[b][i] = j < end && sees(p, j, t.window, two) ? s[b][i] : kNegInf;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < kNB; b++)
#pragma unroll
      for (int i = 0; i < kC; i++) top = fmaxf(top, s[b][i]);
    top *= mul;
    if (__ballot(top > m + kLag)) {
#pragma unroll
      for (int w = MF; w < 64; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
      const float next = fmaxf(m, top);
      const float old = __builtin_amdgcn_exp2f(m - (next == kNegInf ? 0.0f : next));
      m = next;
      l *= old;
#pragma unroll
      for (int d = 0; d < kND; d++)
#pragma unroll
        for (int i = 0; i < kC; i++) o[d][i] *= old;
    }
    const float ref = (m == kNegInf ? 0.0f : m) - kLift;
    // Steps of 8 (binary32: 4) registers of a lane's scores.  A step's products run while the
    // next one's weights are computed and its values read.
    constexpr int kRegs = sizeof(T) == 2 ? 8 : 4, kSteps = kNB * kC / kRegs;
    frag w[2][Op::kTerms], v[2][kVals];
    auto weights = [&](int st) {
      float e[kRegs];
#pragma unroll
      for (int i = 0; i < kRegs; i++) {
        const int r = st * kRegs + i;
        e[i] = __builtin_amdgcn_exp2f(fmaf(s[r / kC][r % kC], mul, -ref));
        l += e[i];
      }
      Op::split(e, w[st & 1]);
    };
    const ValuesAt at = values_at(vd);
    read_values(at, 0, v[0]);
    weights(0);
#pragma unroll
    for (int st = 0; st < kSteps; st++) {
      if (st + 1 < kSteps) {
        if constexpr (!DMA) read_values(at, st + 1, v[(st + 1) & 1]);
        weights(st + 1);
      }
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = 0; k < Op::kTerms; k++)
#pragma unroll
          for (int d = 0; d < kND; d++) mfma<MF>(v[st & 1][d], w[st & 1][k], o[d]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int d = 0; d < kND; d++) mfma<MF>(v[st & 1][d][i], w[st & 1][0][i], o[d]);
      }
      if constexpr (DMA) {
        if (st + 1 < kSteps) read_values(at, st + 1, v[(st + 1) & 1]);
      }
    }
  }

  // Where a lane reads values, and the operand of step st: key_of's order of keys.
  struct ValuesAt {
    uint32_t row, x;
    const char *base;
  };
  static __device__ __forceinline__ ValuesAt values_at(const char *vd) {
    const int lane = threadIdx.x & 63, c = lane % MF, kg = lane / MF;
    if constexpr (sizeof(T) == 2) {
      const int g = lane >> 4, i16 = lane & 15, half = MF == 32 ? g & 1 : 0;
      const uint32_t row = (4 * kg + (i16 >> 2)) * R::kBytes + 8 * (i16 & 1);
      const int swz = R::swz_v(4 * kg + (i16 >> 2));
      return {row, (uint32_t)((2 * half + ((i16 & 3) >> 1)) ^ swz) << 4, vd};
    } else {
      return {(uint32_t)(4 * kg * R::kBytes + (c & 3) * 4),
              (uint32_t)((c >> 2) ^ R::swz_v(4 * kg)) << 4, vd};
    }
  }
  static __device__ __forceinline__ void read_values(const ValuesAt &y, int st,
                                                     frag (&v)[kVals]) {
    if constexpr (sizeof(T) == 2) {
      constexpr int kKeys = 8 * kG, kN = kND > 4 ? kND / 2 : kND;
      const uint32_t off = st * kKeys * R::kBytes;
      if constexpr (DMA) {
#pragma unroll
        for (int d0 = 0; d0 < kND; d0 += kN) {
          uint32_t at[kN];
          s4vec lo[kN], hi[kN];
#pragma unroll
          for (int d = 0; d < kN; d++)
            at[d] = lds_addr(y.base) + off + y.row + (y.x ^ (uint32_t)((d0 + d) * (MF / 8) << 4));
          lds_tr<0, kKeys / 2 * R::kBytes>(at, lo, hi);
#pragma unroll
          for (int d = 0; d < kN; d++) v[d0 + d] = join(lo[d], hi[d]);
        }
      } else {
#pragma unroll
        for (int d = 0; d < kND; d++) {
          const char *at = y.base + y.row + (y.x ^ (uint32_t)(d * (MF / 8) << 4)) + off;
          v[d] = join(lds_tr4(at), lds_tr4(at + kKeys / 2 * R::kBytes));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = 4 * st + i, key = key_of(r / kC, r % kC);
#pragma unroll
        for (int d = 0; d < kND; d++)
          v[d][i] = *(const float *)(y.base + y.row + (y.x ^ d * (MF / 4) << 4) +
                                     key * R::kBytes);
      }
    }
  }
  static __device__ __forceinline__ frag join(s4vec lo, s4vec hi) {
    struct {
      s4vec a, b;
    } v = {lo, hi};
    return __builtin_bit_cast(frag, v);
  }

  // Another wave's sums of the same rows over other keys: put() by that wave, add() by this one,
  // through kPutBytes of LDS.
  static constexpr int kPutBytes = (kND * kC + 2) * 256;
  __device__ __forceinline__ void put(char *lds) const {
    float *to = (float *)lds + (threadIdx.x & 63);
#pragma unroll
    for (int d = 0; d < kND; d++)
#pragma unroll
      for (int i = 0; i < kC; i++) to[(d * kC + i) * 64] = o[d][i];
    to[kND * kC * 64] = m;
    to[(kND * kC + 1) * 64] = l;
  }
  __device__ __forceinline__ void add(const char *lds) {
    const float *from = (const float *)lds + (threadIdx.x & 63);
    const float m2 = from[kND * kC * 64], next = fmaxf(m, m2);
    const float ref = next == kNegInf ? 0.0f : next;
    const float f = __builtin_amdgcn_exp2f(m - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
    m = next;
    l = l * f + from[(kND * kC + 1) * 64] * f2;
#pragma unroll
    for (int d = 0; d < kND; d++)
#pragma unroll
      for (int i = 0; i < kC; i++) o[d][i] = o[d][i] * f + from[(d * kC + i) * 64] * f2;
  }

  // Joins the lane groups' sums; whether the lane's row is finite.
  __device__ __forceinline__ bool end() {
    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // 0, or NaN with a sum that is not finite
#pragma unroll
    for (int d = 0; d < kND; d++)
#pragma unroll
      for (int i = 0; i < kC; i++) z[i & 3] = fmaf(o[d][i], 0.0f, z[i & 3]);
    l += z[0] + z[1] + (z[2] + z[3]);
#pragma unroll
    for (int w = MF; w < 64; w *= 2) l += __shfl_xor(l, w);
    return paged_finite(l);
  }
  // The lane's values of its row times `mul`, to `to` (hd values, any float's address).
  __device__ __forceinline__ void store(float *to, int hd, float mul) const {
    const int kg = ((int)threadIdx.x & 63) / MF;
    auto put = [&](bool all) {
#pragma unroll
      for (int d = 0; d < kND; d++)
#pragma unroll
        for (int i = 0; i < kC; i += 4) {
          const int at = d * MF + key_of(0, i) + 4 * kg;
          if (all || at < hd)
            *(f4a4 *)(to + at) = f4a4{o[d][i] * mul, o[d][i + 1] * mul, o[d][i + 2] * mul,
                                      o[d][i + 3] * mul};
        }
    };
    if (hd == HD) put(true);
    else put(false);
  }
};

}  // namespace mmnb
