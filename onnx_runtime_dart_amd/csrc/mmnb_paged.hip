// Paged key/value cache: storing a batch's new rows, and the entry points.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mmnb_paged.h"

namespace mmnb {

// ---------------------------------------------------------------------------
// Append.  A token's H query heads, G key heads and G value heads are cut into
// items that a thread handles alone, reading all of an item before it writes,
// so that queries may be turned in place: N rotary pairs, or 2 N values that
// pass through.  Rotation in double (two products cancel), rounded to binary32 and
// then to the cache's type.  Bound by memory: 30001 rows of 32 + 16 heads of 128 (0.78 GB fetched,
// 0.61 written) 268 us, 5.2 TB/s; 4 rows 5.6 us, of which 3.6 are the kernel's.
// ---------------------------------------------------------------------------
struct AppendArgs {
  const float *q, *k, *v, *cos, *sin;
  float *qo;
  int64_t ldq, ldk, ldv, ldqo;
  int heads, max_pos, half, first;
};

// The entries of start[0 .. batch] at or below t.  Counted by the whole workgroup in one round of
// loads per 256 sequences, which for a few hundred of them is one memory latency where a binary
// search is eight.
__device__ __forceinline__ int starts_upto(const PagedArgs &a, int t) {
  int n = 0;
  for (int b = 0; b <= a.batch; b += blockDim.x) {
    const int i = b + threadIdx.x;
    n += __syncthreads_count(i <= a.batch && a.start[i] <= t);
  }
  return n;
}

// Where the two halves (N values each) of item i of a head lie.  Pairs come first, then what
// passes through.
struct AppendItem {
  int d0, d1;
  bool turn;
};
template <int N, bool INTER>
__device__ __forceinline__ AppendItem append_item(int i, int half) {
  const int pairs = half / N;
  if (i >= pairs) {
    const int d = 2 * half + (i - pairs) * 2 * N;
    return {d, d + N, false};
  }
  if constexpr (INTER) return {2 * N * i, 2 * N * i + N, true};
  return {N * i, half + N * i, true};
}

// N values of a row, from any float's address.
template <int N>
__device__ __forceinline__ void load_row(const float *p, float (&x)[N]) {
  if constexpr (N == 4) {
    const f4a4 v = *(const f4a4 *)p;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = v[i];
  } else {
    x[0] = p[0];
  }
}
template <int N>
__device__ __forceinline__ void store_row(float *p, const float (&x)[N]) {
  if constexpr (N == 4) {
    *(f4a4 *)p = f4a4{x[0], x[1], x[2], x[3]};
  } else {
    p[0] = x[0];
  }
}
// ... to the cache: rows are aligned to 16 bytes and p to N values of them.
template <int N, typename T>
__device__ __forceinline__ void store_cache(T *p, const float (&x)[N]) {
  if constexpr (N == 4) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    *(v4 *)p = v4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
  } else {
    p[0] = (T)x[0];
  }
}

template <int N, bool INTER>
__device__ __forceinline__ void turn(float (&x)[N], float (&y)[N], const float (&c)[N],
                                     const float (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    // pair i: (x[i], y[i]), or the neighbours 2i and 2i + 1 of x then y
    float &u = INTER ? (2 * i < N ? x[2 * i] : y[2 * i - N]) : x[i];
    float &w = INTER ? (2 * i + 1 < N ? x[2 * i + 1] : y[2 * i + 1 - N]) : y[i];
    const double a = u, b = w, cd = c[i], sd = s[i];
    u = (float)(a * cd - b * sd);
    w = (float)(b * cd + a * sd);
  }
}

template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(256) k_paged_append(PagedArgs a, AppendArgs p) {
  const int t = blockIdx.x, n = starts_upto(a, t);
  if (n == 0 || n > a.batch) return;
  int b = n - 1;  // the last one to begin at or before t: the row's where starts rise
  PagedSeq s = seq_of(a, b);
  if (!paged_in(s, t)) {
    b = scan_for_row(a, t);
    if (b < 0) return;
    s = seq_of(a, b);
  }
  const bool fine = !s.bad;
  const int j = fine ? s.len - s.n + (t - s.row0) : 0;  // key
  const bool past = !fine || p.first + j >= p.max_pos;  // of the tables: NaN
  bool lost = !fine;
  int64_t at = 0;
  if (fine) {
    const int page = paged_page(a.pages[b * a.cols + (j >> a.shift)], a.num_pages, &lost);
    at = row_at(a, page, 0, 0, j);
  }
  const int pairs = p.half / N, per = pairs + (a.hd - 2 * p.half) / (2 * N);
  const int nq = p.q ? p.heads : 0, all = (nq + 2 * a.kv_heads) * per;
  const int it = blockIdx.y * blockDim.x + threadIdx.x;
  if (it >= all) return;
  const int head = it / per;
  const AppendItem e = append_item<N, INTER>(it % per, p.half);
  const bool is_q = head < nq, is_v = head >= nq + a.kv_heads;
  const int g = head - (is_q ? 0 : is_v ? nq + a.kv_heads : nq);
  const float *src = (is_q ? p.q + t * p.ldq : is_v ? p.v + t * p.ldv : p.k + t * p.ldk) +
                     (int64_t)g * a.hd;
  float x[N], y[N];
  load_row<N>(src + e.d0, x);
  load_row<N>(src + e.d1, y);
  if (e.turn && !is_v) {
    const int64_t angle = (int64_t)(past ? 0 : p.first + j) * p.half + N * (it % per);
    float co[N], si[N];
    load_row<N>(p.cos + angle, co);
    load_row<N>(p.sin + angle, si);
    turn<N, INTER>(x, y, co, si);
#pragma unroll
    for (int i = 0; i < N; i++) {
      x[i] = past ? __builtin_nanf("") : x[i];
      y[i] = past ? __builtin_nanf("") : y[i];
    }
  }
  if (is_q) {
    float *to = p.qo + t * p.ldqo + (int64_t)g * a.hd;
    if (!fine) {
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = y[i] = __builtin_nanf("");
    }
    store_row<N>(to + e.d0, x);
    store_row<N>(to + e.d1, y);
  } else if (!lost) {
    T *to = (T *)(is_v ? a.v : a.k) + at + g * a.sh;
    store_cache<N, T>(to + e.d0, x);
    store_cache<N, T>(to + e.d1, y);
  }
}

// ---------------------------------------------------------------------------
// Items of four pairs where the pairs are a multiple of four, else of one (a pair of values
// that passes through counts as one too).
template <typename T, int N, bool INTER>
static int launch_append(mmnb_ctx *ctx, const PagedArgs &a, const AppendArgs &p) {
  const int64_t items = (int64_t)((p.q ? p.heads : 0) + 2 * a.kv_heads) *
                        (p.half / N + (a.hd - 2 * p.half) / (2 * N));
  // workgroups of equal size, 256 threads at most
  const int64_t parts = (items + 255) / 256, threads = ((items + parts - 1) / parts + 63) / 64 * 64;
  return launch(ctx, kKernPagedAppend, k_paged_append<T, N, INTER>,
                dim3((unsigned)a.tokens, (unsigned)parts), dim3((unsigned)threads), 0, a, p);
}
template <typename T>
static int launch_append(mmnb_ctx *ctx, const PagedArgs &a, const AppendArgs &p, bool inter) {
  if (p.half % 4 == 0)
    return inter ? launch_append<T, 4, true>(ctx, a, p) : launch_append<T, 4, false>(ctx, a, p);
  return inter ? launch_append<T, 1, true>(ctx, a, p) : launch_append<T, 1, false>(ctx, a, p);
}

static int run_attention(mmnb_ctx *ctx, const char *op, const mmnb_paged_cache *cache,
                         const mmnb_paged_batch *batch, const int32_t *d_prefix_pages,
                         int64_t prefix_len, const mmnb_paged_scores *scores, const float *d_q,
                         int64_t ldq, int64_t num_heads, float *d_out, int64_t ldo) {
  MMNB_PAGED(op, paged_check_cache(cache));
  MMNB_PAGED(op, paged_check_batch(*cache, batch));
  MMNB_PAGED(op, paged_check_rows(*cache, num_heads, ldq));
  MMNB_PAGED(op, paged_check_rows(*cache, num_heads, ldo));
  MMNB_PAGED(op, paged_check_heads(*cache, num_heads));
  MMNB_PAGED(op, paged_check_size(*batch, num_heads));
  MMNB_PAGED(op, paged_check_scores(scores));
  MMNB_PAGED(op, paged_check_prefix(*batch, d_prefix_pages, prefix_len));
  if (batch->batch == 0 || batch->tokens == 0) return MMNB_OK;
  if (!d_q || !d_out) return refuse(op, paged_arg("null buffer"));
  const PagedArgs a = paged_args(*cache, *batch);
  AttnArgs t = {};
  t.q = d_q, t.ldq = ldq, t.out = d_out, t.ldo = ldo;
  t.heads = (int)num_heads, t.group = (int)(num_heads / cache->kv_heads);
  t.inv_group = 1.0f / (float)t.group;
  t.ppages = d_prefix_pages, t.prefix = (int)prefix_len;
  const PagedFactors f = paged_factors(scores, cache->head_size);
  t.capped = f.capped, t.mul = f.mul, t.in_mul = f.in_mul;
  // (a window that reaches past every key is none)
  t.window = scores && scores->window < prefix_len + batch->max_kv ? (int)scores->window : 0;
  t.slopes = scores ? scores->d_slopes : nullptr;
  t.two = scores ? scores->d_two_way : nullptr;
  t.seen = paged_prefix_seen(t.prefix, t.window, t.two != nullptr);
  CtxLock lk(ctx);
  int rc = set_device(ctx);
  if (rc) return rc;
  // The first call of any form leaves memory for pieces behind, so that a step may be recorded
  // after, say, a prompt in one part, which needs none itself.  (One that needs them asks again.)
  void *buf;
  if (!ctx->capturing && !ctx->scratch[kPagedScratch].ptr)
    (void)scratch_get(ctx, kPagedScratch, kPagedScratchBytes, &buf);
  switch (cache->type) {
    case MMNB_DT_F32: return paged_attention_f32(ctx, a, t);
    case MMNB_DT_F16: return paged_attention_f16(ctx, a, t);
    default: return paged_attention_bf16(ctx, a, t);
  }
}

}  // namespace mmnb

using namespace mmnb;

extern "C" {

int mmnb_paged_append_dev(mmnb_ctx *ctx, const mmnb_paged_cache *cache,
                          const mmnb_paged_batch *batch, const float *d_q, int64_t ldq,
                          int64_t num_heads, const float *d_k, int64_t ldk, const float *d_v,
                          int64_t ldv, const float *d_cos, const float *d_sin,
                          int64_t max_pos, int64_t half_rot, int interleaved,
                          int64_t first_pos, float *d_q_out, int64_t ldqo) {
  static const char *op = "paged append";
  MMNB_GUARD_CTX(ctx);
  MMNB_PAGED(op, paged_check_cache(cache));
  MMNB_PAGED(op, paged_check_batch(*cache, batch));
  if (d_q) {
    MMNB_PAGED(op, paged_check_rows(*cache, num_heads, ldq));
    MMNB_PAGED(op, paged_check_rows(*cache, num_heads, ldqo));
  }
  MMNB_PAGED(op, paged_check_rows(*cache, cache->kv_heads, ldk));
  MMNB_PAGED(op, paged_check_rows(*cache, cache->kv_heads, ldv));
  MMNB_PAGED(op, paged_check_rope(*cache, *batch, d_cos, d_sin, max_pos, half_rot, first_pos));
  if (batch->batch == 0 || batch->tokens == 0) return MMNB_OK;
  if (!d_k || !d_v || (d_q && !d_q_out)) return refuse(op, paged_arg("null buffer"));
  if (d_q)
    MMNB_PAGED(op, paged_check_in_place(d_q, ldq, d_q_out, ldqo, num_heads * cache->head_size,
                                        batch->tokens));
  const PagedArgs a = paged_args(*cache, *batch);
  AppendArgs p;
  p.q = d_q, p.k = d_k, p.v = d_v, p.cos = d_cos, p.sin = d_sin, p.qo = d_q_out;
  p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.ldqo = ldqo;
  p.heads = (int)num_heads, p.max_pos = (int)std::min<int64_t>(max_pos, INT32_MAX);
  p.half = (int)half_rot, p.first = (int)first_pos;
  CtxLock lk(ctx);
  int rc = set_device(ctx);
  if (rc) return rc;
  switch (cache->type) {
    case MMNB_DT_F32: return launch_append<float>(ctx, a, p, interleaved != 0);
    case MMNB_DT_F16: return launch_append<_Float16>(ctx, a, p, interleaved != 0);
    default: return launch_append<__bf16>(ctx, a, p, interleaved != 0);
  }
}

int mmnb_paged_attention_dev(mmnb_ctx *ctx, const mmnb_paged_cache *cache,
                             const mmnb_paged_batch *batch,
                             const mmnb_paged_scores *scores, const float *d_q, int64_t ldq,
                             int64_t num_heads, float *d_out, int64_t ldo) {
  MMNB_GUARD_CTX(ctx);
  return run_attention(ctx, "paged attention", cache, batch, nullptr, 0, scores, d_q, ldq,
                       num_heads, d_out, ldo);
}

int mmnb_paged_attention_shared_dev(mmnb_ctx *ctx, const mmnb_paged_cache *cache,
                                    const mmnb_paged_batch *batch,
                                    const int32_t *d_prefix_pages, int64_t prefix_len,
                                    const mmnb_paged_scores *scores, const float *d_q,
                                    int64_t ldq, int64_t num_heads, float *d_out,
                                    int64_t ldo) {
  MMNB_GUARD_CTX(ctx);
  return run_attention(ctx, "paged attention (shared prefix)", cache, batch, d_prefix_pages,
                       prefix_len, scores, d_q, ldq, num_heads, d_out, ldo);
}

}  // extern "C"
