// Log-probabilities of given tokens, with the row's entropy and its most
// likely tokens, and the gradient of the first two.
//
// For a row x of V logits and a token t, with m = max x and S = sum exp(x - m):
//
//   log p_i = (x_i - m) - log S          entropy H = log S - (1/S) sum e_i (x_i - m),  e_i = exp(x_i - m)
//   d log p_t / d x_i = [i = t] - p_i    d H / d x_i = -p_i (log p_i + H)
//
// The reference has the parts as separate ops (log_softmax.wgsl, a gather, a
// sum, a sort); this is the one pass over the logits they need.  m and log S
// are kept apart in `stats`: their f32 sum would lose the low bits of log S
// under a large m, and the backward pass takes exp of the difference.
#include <cuda_runtime.h>

#include <cfloat>
#include <climits>

#include "tp_core.h"
#include "tp_launch.h"
#include "tp_token.cuh"

namespace tp {

constexpr int LP_MAX_TOP = 32;

// Order of the alternatives: larger logit first, then the lower index; one
// 64-bit key, larger is better.  Adding 0 makes -0 and 0 the same logit.
__device__ __forceinline__ unsigned long long lp_key(float x, uint32_t i) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)o << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float lp_key_value(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int32_t lp_key_index(unsigned long long k) { return (int32_t)~(uint32_t)k; }

template <class T, class F>
__device__ T lp_block(T v, T* sh, F f) {
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v = f(v, sh[w]);
  return v;
}

__global__ void __launch_bounds__(256) k_logprobs(const float* x, int64_t ld, const void* ids, int kind, int64_t V,
                                                  int K, float* logp, float* entropy, float* stats, int32_t* top_ids,
                                                  float* top_logp) {
  ::tp::pdl_enter();
  __shared__ float shf[8];
  __shared__ unsigned long long shk[8];
  const int64_t row = blockIdx.x;
  const float* xr = x + row * ld;
  auto fmx = [](float a, float b) { return (isnan(a) || a > b) ? a : b; };
  auto fad = [](float a, float b) { return a + b; };
  auto kmx = [](unsigned long long a, unsigned long long b) { return a > b ? a : b; };
  float m = -INFINITY;
  for (int64_t i = threadIdx.x; i < V; i += 256) m = fmx(m, xr[i]);
  m = lp_block(m, shf, fmx);
  const bool none = m == -INFINITY, bad = isnan(m) || m == INFINITY;
  float S = 0.0f, T = 0.0f;
  if (!none && !bad)
    for (int64_t i = threadIdx.x; i < V; i += 256) {
      const float y = xr[i] - m, e = expf(y);
      S += e;
      if (e > 0.0f) T += e * y;
    }
  S = lp_block(S, shf, fad);
  T = lp_block(T, shf, fad);
  const float lnS = none ? -INFINITY : (bad ? NAN : logf(S));
  if (threadIdx.x == 0) {
    if (entropy) entropy[row] = none ? 0.0f : (bad ? NAN : lnS - T / S);
    if (stats) {
      stats[2 * row] = bad ? NAN : m;
      stats[2 * row + 1] = lnS;
    }
    if (logp) {
      const int64_t t = token_id(ids, kind, row);
      logp[row] = t < 0 ? 0.0f : (t >= V || bad ? NAN : (none ? -INFINITY : (xr[t] - m) - lnS));
    }
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < K; ++k) {
    unsigned long long best = 0ull;
    if (!bad && !none)
      for (int64_t i = threadIdx.x; i < V; i += 256) {
        const float v = xr[i];
        const unsigned long long q = v == -INFINITY ? 0ull : lp_key(v, (uint32_t)i);
        if (q < last && q > best) best = q;
      }
    best = lp_block(best, shk, kmx);
    last = best;
    if (threadIdx.x == 0) {
      top_ids[row * K + k] = best ? lp_key_index(best) : -1;
      top_logp[row * K + k] = best ? (lp_key_value(best) - m) - lnS : (bad ? NAN : -INFINITY);
    }
  }
}

__global__ void __launch_bounds__(256) k_logprobs_bwd(const float* x, int64_t ld, const void* ids, int kind,
                                                      const float* stats, const float* entropy, const float* dlogp,
                                                      const float* dentropy, int64_t V, float* dx, int64_t ldd) {
  ::tp::pdl_enter();
  const int64_t row = blockIdx.x;
  const float* xr = x + row * ld;
  float* dr = dx + row * ldd;
  const float m = stats[2 * row], lnS = stats[2 * row + 1];
  const int64_t t = ids ? token_id(ids, kind, row) : -1;
  float c1 = dlogp && t >= 0 ? dlogp[row] : 0.0f, c2 = dentropy ? dentropy[row] : 0.0f;
  if (m == -INFINITY || (c1 == 0.0f && c2 == 0.0f)) {
    for (int64_t i = threadIdx.x; i < V; i += 256) dr[i] = 0.0f;
    return;
  }
  if (isnan(m) || (c1 != 0.0f && t >= V)) c1 = NAN;
  const float H = c2 != 0.0f ? entropy[row] : 0.0f;
  for (int64_t i = threadIdx.x; i < V; i += 256) {
    const float lp = fmaxf((xr[i] - m) - lnS, -1e4f), p = expf(lp);
    dr[i] = c1 * ((i == t ? 1.0f : 0.0f) - p) - c2 * (p * (lp + H));
  }
}

void launch_logprobs(const float* x, int64_t ld, const void* ids, int kind, int64_t R, int64_t V, int K, float* logp,
                     float* entropy, float* stats, int32_t* top_ids, float* top_logp) {
  if (R == 0) return;
  TP_LAUNCH(k_logprobs, (unsigned)R, 256, 0, x, ld, ids, kind, V, K, logp, entropy, stats, top_ids, top_logp);
}

void launch_logprobs_bwd(const float* x, int64_t ld, const void* ids, int kind, const float* stats,
                         const float* entropy, const float* dlogp, const float* dentropy, int64_t R, int64_t V,
                         float* dx, int64_t ldd) {
  if (R == 0) return;
  TP_LAUNCH(k_logprobs_bwd, (unsigned)R, 256, 0, x, ld, ids, kind, stats, entropy, dlogp, dentropy, V, dx, ldd);
}

static void check_logprobs(int64_t R, int64_t V, int64_t ld, const char* what) {
  TP_REQUIRE(R >= 0 && R <= INT_MAX, "%s: %lld rows is outside [0, 2^31)", what, (long long)R);
  check_vocab(V, what);
  TP_REQUIRE(ld >= V, "%s: a row stride of %lld is shorter than the %lld logits of a row", what, (long long)ld,
             (long long)V);
}

static void check_top(int K, int64_t V, const char* what) {
  TP_REQUIRE(K >= 0 && K <= LP_MAX_TOP && K <= V, "%s: topk must be in [0, min(%d, %lld)], got %d", what, LP_MAX_TOP,
             (long long)V, K);
}

}  // namespace tp

using namespace tp;

extern "C" {

TP_API int tpk_token_logprobs(const float* logits, int64_t ld, const void* ids, int ids_kind, int64_t rows,
                              int64_t vocab, int topk, float* logp, float* entropy, float* stats, int32_t* top_ids,
                              float* top_logp) {
  return guard([&] {
    const char* what = "token_logprobs";
    check_logprobs(rows, vocab, ld, what);
    check_top(topk, vocab, what);
    check_ids_kind(ids_kind, what);
    if (rows == 0) return;
    TP_REQUIRE(logits, "%s: logits is NULL", what);
    TP_REQUIRE(!logp || ids, "%s: log-probabilities need token ids", what);
    TP_REQUIRE(topk == 0 || (top_ids && top_logp), "%s: topk > 0 needs both outputs of the alternatives", what);
    TP_REQUIRE(((uintptr_t)logits & 3) == 0, "%s: logits are not 4-byte aligned", what);
    launch_logprobs(logits, ld, ids, ids_kind, rows, vocab, topk, logp, entropy, stats, top_ids, top_logp);
  });
}

TP_API int tpk_token_logprobs_backward(const float* logits, int64_t ld, const void* ids, int ids_kind,
                                       const float* stats, const float* entropy, const float* dlogp,
                                       const float* dentropy, int64_t rows, int64_t vocab, float* dlogits,
                                       int64_t ldd) {
  return guard([&] {
    const char* what = "token_logprobs_backward";
    check_logprobs(rows, vocab, ld, what);
    check_logprobs(rows, vocab, ldd, what);
    check_ids_kind(ids_kind, what);
    if (rows == 0) return;
    TP_REQUIRE(logits && stats && dlogits, "%s: logits, stats and dlogits must not be NULL", what);
    TP_REQUIRE(!dlogp || ids, "%s: a gradient of log-probabilities needs token ids", what);
    TP_REQUIRE(!dentropy || entropy, "%s: a gradient of the entropy needs the entropy", what);
    TP_REQUIRE((((uintptr_t)logits | (uintptr_t)dlogits) & 3) == 0, "%s: a buffer is not 4-byte aligned", what);
    TP_REQUIRE(dlogits != logits || ldd == ld, "%s: in place needs the same row stride", what);
    launch_logprobs_bwd(logits, ld, ids, ids_kind, stats, entropy, dlogp, dentropy, rows, vocab, dlogits, ldd);
  });
}

TP_API int tp_token_logprobs(int64_t logits, int64_t ids, int topk, tp_handle* logp, tp_handle* entropy,
                             tp_handle* stats, tp_handle* top_ids, tp_handle* top_logp) {
  return guard([&] {
    const char* what = "tokenLogprobs";
    const Tensor X = get(logits), I = get(ids);
    TP_REQUIRE(X.ndim >= 1 && X.phys == PHYS_F32, "%s: expects float logits [..., vocab]", what);
    const int64_t V = X.shape[X.ndim - 1];
    check_vocab(V, what);
    const int64_t R = X.numel / V;
    TP_REQUIRE(I.numel == R, "%s: %lld token ids for %lld rows of logits", what, (long long)I.numel, (long long)R);
    check_logprobs(R, V, V, what);
    check_top(topk, V, what);
    TP_REQUIRE(topk == 0 || I.ndim < TP_MAX_DIMS, "%s: ids of rank %d leave no dim for the alternatives", what, I.ndim);
    TP_REQUIRE(I.ndim < TP_MAX_DIMS, "%s: ids of rank %d leave no dim for the statistics", what, I.ndim);
    std::vector<int64_t> s = shape_of(I), s2 = s, sk = s;
    s2.push_back(2);
    sk.push_back(topk);
    Outputs o;
    Tensor &lp = o.add(make_like_shape(s, X.dtype)), &en = o.add(make_like_shape(s, X.dtype));
    Tensor &st = o.add(make_like_shape(s2, X.dtype)), &ti = o.add(make_like_shape(sk, TP_INT64, PHYS_I32));
    Tensor& tl = o.add(make_like_shape(sk, X.dtype));
    launch_logprobs(X.f(), V, I.ptr, ids_kind_of(I), R, V, topk, lp.f(), en.f(), st.f(), ti.i(), tl.f());
    o.emit_all({logp, entropy, stats, top_ids, top_logp});
  });
}

TP_API int tp_token_logprobs_backward(int64_t dlogp, int64_t dentropy, int64_t logits, int64_t ids, int64_t stats,
                                      int64_t entropy, tp_handle* out) {
  return guard([&] {
    const char* what = "tokenLogprobsBackward";
    const Tensor X = get(logits), I = get(ids), St = get(stats), En = get(entropy);
    TP_REQUIRE(X.ndim >= 1 && X.phys == PHYS_F32, "%s: expects float logits [..., vocab]", what);
    const int64_t V = X.shape[X.ndim - 1];
    check_vocab(V, what);
    const int64_t R = X.numel / V;
    TP_REQUIRE(I.numel == R && St.numel == 2 * R && En.numel == R,
               "%s: ids, stats and entropy do not belong to %lld rows of logits", what, (long long)R);
    const Tensor g1 = dlogp ? get(dlogp) : Tensor(), g2 = dentropy ? get(dentropy) : Tensor();
    TP_REQUIRE((!dlogp || g1.numel == R) && (!dentropy || g2.numel == R),
               "%s: a gradient does not have %lld values", what, (long long)R);
    TP_REQUIRE(g1.phys == PHYS_F32 && g2.phys == PHYS_F32 && St.phys == PHYS_F32 && En.phys == PHYS_F32,
               "%s: index tensors are not supported as gradients or statistics", what);
    check_logprobs(R, V, V, what);
    Outputs o;
    Tensor& d = o.add(make(X.shape, X.ndim, X.dtype));
    launch_logprobs_bwd(X.f(), V, I.ptr, ids_kind_of(I), St.f(), En.f(), dlogp ? g1.f() : nullptr,
                        dentropy ? g2.f() : nullptr, R, V, d.f(), V);
    o.emit_all({out});
  });
}

}  // extern "C"
