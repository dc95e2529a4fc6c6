// Device side of the paged key/value cache: what its kernels share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "mmnb_internal.h"
#include "mmnb_paged_plan.h"

namespace mmnb {

// A call's cache and batch, as every kernel of it takes them.
struct PagedArgs {
  const char *k, *v;             // append writes through them
  int64_t sp, sh, sr;            // strides, elements
  int num_pages, shift;          // page_size = 1 << shift
  const int32_t *start, *kv_len, *pages;
  int64_t cols;
  int batch, tokens, max_q, max_kv;
  int kv_heads, hd;
};

// What attention takes besides.
struct AttnArgs {
  const float *q;
  int64_t ldq;
  float *out;
  int64_t ldo;
  int heads, group;
  float inv_group;               // 1 / group
  const int32_t *ppages;         // shared prefix of `prefix` keys
  int prefix;
  int seen;                      // no row sees a prefix key below it (a multiple of 64)
  // scores in base 2: z2 = mul dot, or with a cap mul tanh(dot in_mul)
  float mul, in_mul;
  int capped;
  int window;                    // 0: none
  const float *slopes;
  const int32_t *two;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

// ---- the cache's types
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));  // any float's address

template <typename T>
__device__ __forceinline__ float widen(T x) {
  return (float)x;
}

// Eight values from an address aligned to 16 bytes.
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
  const f4 a = *(const f4 *)p, b = *(const f4 *)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
}
__device__ __forceinline__ void load8(const _Float16 *p, float (&x)[8]) {
  const half8 a = *(const half8 *)p;
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = (float)a[i];
}
__device__ __forceinline__ void load8(const __bf16 *p, float (&x)[8]) {
  const bf8 a = *(const bf8 *)p;
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = (float)a[i];
}

// ---- sequences and keys
__device__ __forceinline__ PagedSeq seq_of(const PagedArgs &a, int b) {
  return paged_seq(a.start[b], a.start[b + 1], a.kv_len[b], a.tokens, a.max_q, a.max_kv);
}

// The first sequence that holds row t (-1: none), by a wave that looks at all of them: for
// batches whose starts do not rise, and rows of no sequence.
__device__ __forceinline__ int scan_for_row(const PagedArgs &a, int t) {
  for (int c = 0; c < a.batch; c += 256) {
    bool in[4];  // four rounds of loads at once
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int i = c + 64 * u + ((int)threadIdx.x & 63);
      in[u] = i < a.batch && paged_holds(a.start, i, t);
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const uint64_t any = __ballot(in[u]);
      if (any) return c + 64 * u + __builtin_ctzll(any);
    }
  }
  return -1;
}

// The page of key j of a sequence: of the shared prefix below `prefix`, of its own from there
// on.  Sets *bad for a number outside the cache (and gives page 0).
__device__ __forceinline__ int page_of(const PagedArgs &a, const int32_t *table,
                                       const int32_t *ppages, int prefix, int j, bool *bad) {
  const int e = j < prefix ? ppages[j >> a.shift] : table[(j - prefix) >> a.shift];
  return paged_page(e, a.num_pages, bad);
}
// Elements from the cache's begin to key j's row of head g in `page`.
__device__ __forceinline__ int64_t row_at(const PagedArgs &a, int page, int prefix, int g, int j) {
  const int r = (j < prefix ? j : j - prefix) & ((1 << a.shift) - 1);
  return page * a.sp + g * a.sh + r * a.sr;
}

// ---- scores
// Whether the row at position p sees key j (both counted from the prefix's begin); `two` keys
// are seen by every row.
__device__ __forceinline__ bool sees(int p, int j, int window, int two) {
  return (j <= p && (window == 0 || p - j < window)) || j < two;
}

// tanh to about a unit in the last place.  Small arguments: the quotient's form loses what
// cancels in it, so the odd series up to x^13 (its next term is below 2^-25 x there).
__device__ __forceinline__ float paged_tanh(float x) {
  const float a = fabsf(x);
  const float e = __builtin_amdgcn_exp2f(2.0f * kLog2e * a);  // may be infinite
  const float far = fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
  const float s = x * x;
  float t = 21844.0f / 6081075.0f;
  t = fmaf(t, s, -1382.0f / 155925.0f);
  t = fmaf(t, s, 62.0f / 2835.0f);
  t = fmaf(t, s, -17.0f / 315.0f);
  t = fmaf(t, s, 2.0f / 15.0f);
  t = fmaf(t, s, -1.0f / 3.0f);
  const float near = fmaf(x * s, t, x);
  return a < 0.35f ? near : copysignf(far, x);
}

// The score in base 2 of a product q.k; slope is the head's, in base 2.
__device__ __forceinline__ float score2(const AttnArgs &t, float dot, float slope, int p, int j) {
  const float z = t.capped ? t.mul * paged_tanh(dot * t.in_mul) : t.mul * dot;
  return t.slopes ? z - slope * (float)(p < j ? j - p : p - j) : z;
}

// Row and head of the group of row k < 2^21 of a sequence's rows and a head's group in one line:
// the quotient lies at least 1 / (2 group) from a whole number, the product's error below that.
struct GroupRow {
  int i, r;
};
__device__ __forceinline__ GroupRow group_row(const AttnArgs &t, int k) {
  const int i = (int)(((float)k + 0.5f) * t.inv_group);
  return {i, k - i * t.group};
}

// ---- one row, exactly as defined
// Softmax state of one row over keys [lo, hi), by one wave: keys that the row does not see are
// never touched, so nothing in them reaches it, and infinities and NaN in the others act as
// they do in the formula.  Lane l ends with m and l (equal in all lanes) and the sums of
// dimensions l and l + 64.  q: the row's query (uniform).  table: the sequence's pages.
struct RowState {
  float m, l, o0, o1;
};
template <typename T>
__device__ RowState row_exact(const PagedArgs &a, const AttnArgs &t, const int32_t *table,
                              const float *q, int h, int p, int two, int lo, int hi) {
  const int lane = threadIdx.x & 63, g = h / t.group;
  const T *kc = (const T *)a.k, *vc = (const T *)a.v;
  const float slope = t.slopes ? t.slopes[h] * kLog2e : 0.0f;
  RowState s = {kNegInf, 0.0f, 0.0f, 0.0f};
  for (int base = lo; base < hi; base += 64) {
    const int j = base + lane;
    const bool seen = j < hi && sees(p, j, t.window, two);
    uint64_t any = __ballot(seen);
    if (!any) continue;
    float z = kNegInf;
    int64_t at = 0;
    if (seen) {
      bool bad = false;
      const int page = page_of(a, table, t.ppages, t.prefix, j, &bad);
      at = row_at(a, page, t.prefix, g, j);
      float dot = 0.0f;
      for (int d = 0; d < a.hd; d += 8) {
        float x[8];
        load8(kc + at + d, x);
#pragma unroll
        for (int i = 0; i < 8; i++) dot = fmaf(q[d + i], x[i], dot);
      }
      z = bad ? __builtin_nanf("") : score2(t, dot, slope, p, j);
    }
    float top = z;
#pragma unroll
    for (int w = 1; w < 64; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
    const float m = fmaxf(s.m, top), ref = m == kNegInf ? 0.0f : m;
    const float e = seen ? __builtin_amdgcn_exp2f(z - ref) : 0.0f;
    float sum = e;
#pragma unroll
    for (int w = 1; w < 64; w *= 2) sum += __shfl_xor(sum, w);
    const float old = __builtin_amdgcn_exp2f(s.m - ref);
    s.m = m;
    s.l = s.l * old + sum;
    s.o0 *= old;
    s.o1 *= old;
    while (any) {
      const int i = __builtin_ctzll(any);
      any &= any - 1;
      const float w = __shfl(e, i);
      const int64_t r = __shfl(at, i);
      if (lane < a.hd) s.o0 = fmaf(w, widen(vc[r + lane]), s.o0);
      if (lane + 64 < a.hd) s.o1 = fmaf(w, widen(vc[r + lane + 64]), s.o1);
    }
  }
  return s;
}

// ---- host side
constexpr int kPagedScratch = 11;  // the context's slot for pieces of attention's rows
constexpr size_t kPagedScratchBytes = size_t(64) << 20;

int paged_attention_f32(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t);
int paged_attention_f16(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t);
int paged_attention_bf16(mmnb_ctx *ctx, const PagedArgs &a, const AttnArgs &t);

inline int refuse(const char *op, const PagedCheck &c) {
  return fail(c.code, std::string(op) + ": " + c.what);
}
#define MMNB_PAGED(op, check)                             \
  do {                                                    \
    const PagedCheck _c = (check);                        \
    if (_c.code != MMNB_OK) return refuse(op, _c);        \
  } while (0)

inline PagedArgs paged_args(const mmnb_paged_cache &c, const mmnb_paged_batch &b) {
  PagedArgs a;
  const PagedStrides s = paged_strides(c);
  a.k = (const char *)c.k;
  a.v = (const char *)c.v;
  a.sp = s.page, a.sh = s.head, a.sr = s.row;
  a.num_pages = (int)c.num_pages;
  a.shift = __builtin_ctzll((unsigned long long)c.page_size);
  a.start = b.d_start, a.kv_len = b.d_kv_len, a.pages = b.d_pages;
  a.cols = b.page_cols;
  a.batch = (int)b.batch, a.tokens = (int)b.tokens;
  a.max_q = (int)b.max_q, a.max_kv = (int)b.max_kv;
  a.kv_heads = (int)c.kv_heads, a.hd = (int)c.head_size;
  return a;
}

}  // namespace mmnb
