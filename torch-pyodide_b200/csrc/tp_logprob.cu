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

constexpr float LP_L2E = 1.4426950408889634f;
// Differences from the maximum are taken no lower than this: exp is 0 there, and
// 0 * LP_FLOOR is 0 where 0 * -inf (a masked logit, or one so far down that the
// difference overflows) would be NaN.
constexpr float LP_FLOOR = -1e4f;

// exp(y) of y <= 0: one product, one MUFU.  Results below 2^-126 are flushed.
__device__ __forceinline__ float lp_exp(float y) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y * LP_L2E));
  return e;
}
// max that keeps a NaN
__device__ __forceinline__ float lp_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Running statistics of a set of logits: maximum m, S = sum exp(x - m) and
// T = sum exp(x - m) (x - m).  Moving the reference from m to M >= m, with
// d = m - M: S' = exp(d) S, T' = exp(d) (T + d S).
struct LpStat {
  float m, S, T;
  __device__ __forceinline__ void move(float M) {
    const float d = fmaxf(m - M, LP_FLOOR), s = lp_exp(d);
    T = s * fmaf(d, S, T);
    S *= s;
    m = M;
  }
  __device__ __forceinline__ void add(float x) {
    const float y = fmaxf(x - m, LP_FLOOR), e = lp_exp(y);
    S += e;
    T = fmaf(e, y, T);
  }
};

// What a finished row writes; stat: over the whole row.  none: nothing but -inf.
struct LpRow {
  bool none, bad;
  float m, lnS;
  __device__ LpRow(const LpStat& s)
      : none(s.m == -INFINITY), bad(isnan(s.m) || s.m == INFINITY), m(bad ? NAN : s.m),
        lnS(none ? -INFINITY : (bad ? NAN : logf(s.S))) {}
  __device__ void write(const LpStat& s, int64_t row, int64_t V, int t, float xt, float* logp, float* entropy,
                        float* stats) const {
    if (entropy) entropy[row] = none ? 0.0f : (bad ? NAN : lnS - s.T / s.S);
    if (stats) {
      stats[2 * row] = m;
      stats[2 * row + 1] = lnS;
    }
    if (logp) logp[row] = t < 0 ? 0.0f : (t >= V || bad ? NAN : (none ? -INFINITY : (xt - m) - lnS));
  }
  // the k-th alternative from its key (0: there is none)
  __device__ void write_top(unsigned long long key, int64_t at, int32_t* ids, float* lps) const {
    ids[at] = key && !bad ? lp_key_index(key) : -1;
    lps[at] = bad ? NAN : (key ? (lp_key_value(key) - m) - lnS : -INFINITY);
  }
};

// ---- short rows: a warp each, the row in registers ---------------------------------------
// A warp takes `per` rows (at most 8) one after the other; lane r keeps row r's
// statistics, so that logarithms and stores are done for all rows at once.  Lane l
// holds the logits l + 32 k, k < N, of the row at hand and the best two of them.
// The alternatives are found one by one: the warp's largest value, the lowest
// index that has it; the lane it came from puts its second best in its place, or
// looks for it when that is used up too.
constexpr int LP_ROWS = 8;

template <int N, bool TOP>
__global__ void __launch_bounds__(256) k_logprobs_warp(const float* __restrict__ x, int64_t ld,
                                                       const void* __restrict__ ids, int kind, int64_t R, int V,
                                                       int per, int K, float* __restrict__ logp,
                                                       float* __restrict__ entropy, float* __restrict__ stats,
                                                       int32_t* __restrict__ top_ids, float* __restrict__ top_logp) {
  ::tp::pdl_enter();
  __shared__ unsigned long long keys[8][TOP ? LP_ROWS * LP_MAX_TOP : 1];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t row0 = ((int64_t)blockIdx.x * 8 + w) * per;
  if (row0 >= R) return;
  const int rows = R - row0 < per ? (int)(R - row0) : per;
  int t = -1;
  if (logp && lane < rows) t = token_id(ids, kind, row0 + lane);
  LpStat mine{-INFINITY, 0.0f, 0.0f};
  for (int r = 0; r < rows; ++r) {
    const float* __restrict__ xr = x + (row0 + r) * ld;
    float v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = lane + 32 * k;
      v[k] = i < V ? xr[i] : -INFINITY;
    }
    LpStat s{-INFINITY, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < N; ++k) s.m = lp_max(s.m, v[k]);
    for (int o = 16; o > 0; o >>= 1) s.m = lp_max(s.m, __shfl_xor_sync(0xffffffffu, s.m, o));
#pragma unroll
    for (int k = 0; k < N; ++k) s.add(v[k]);
    for (int o = 16; o > 0; o >>= 1) {
      s.S += __shfl_xor_sync(0xffffffffu, s.S, o);
      s.T += __shfl_xor_sync(0xffffffffu, s.T, o);
    }
    if (lane == r) mine = s;
    if (TOP) {
      unsigned long long* out = keys[w] + r * K;
      float b1 = -INFINITY, b2 = -INFINITY;
      int i1 = 0, i2 = 0;
      auto see = [&](float y, int k) {
        if (y > b1) {
          b2 = b1, i2 = i1;
          b1 = y, i1 = k;
        } else if (y > b2) {
          b2 = y, i2 = k;
        }
      };
#pragma unroll
      for (int k = 0; k < N; ++k) see(v[k], k);
      bool second = true;
      const bool odd = !(s.m < INFINITY);  // NaN or +inf in the row: no alternatives
      for (int q = 0; q < K; ++q) {
        const uint32_t o = odd || b1 == -INFINITY ? 0u : (uint32_t)(lp_key(b1, 0) >> 32);
        const uint32_t top = __reduce_max_sync(0xffffffffu, o);
        const uint32_t i = o == top ? (uint32_t)(lane + 32 * i1) : UINT_MAX;
        const uint32_t first = __reduce_min_sync(0xffffffffu, i);
        if (lane == 0) out[q] = top ? (unsigned long long)top << 32 | (uint32_t)~first : 0ull;
        if (top && i == first) {
          if (second) {
            b1 = b2, i1 = i2;
            second = false;
          } else {
            const float y0 = b1;
            const int k0 = i1;
            b1 = b2 = -INFINITY;
#pragma unroll
            for (int k = 0; k < N; ++k)
              if (v[k] < y0 || (v[k] == y0 && k > k0)) see(v[k], k);
            second = true;
          }
        }
      }
    }
  }
  const LpRow a(mine);
  if (lane < rows) {
    const float xt = t >= 0 && t < V ? x[(row0 + lane) * ld + t] : 0.0f;
    a.write(mine, row0 + lane, V, t, xt, logp, entropy, stats);
  }
  if (TOP) {
    __syncwarp();
    for (int e0 = 0; e0 < rows * K; e0 += 32) {
      const int e = e0 + lane, r = e / K;
      LpRow b = a;
      b.bad = __shfl_sync(0xffffffffu, (int)a.bad, r & 31);
      b.m = __shfl_sync(0xffffffffu, a.m, r & 31);
      b.lnS = __shfl_sync(0xffffffffu, a.lnS, r & 31);
      if (e < rows * K) b.write_top(keys[w][e], row0 * K + e, top_ids, top_logp);
    }
  }
}

// ---- long rows: a CTA, or a cluster of CTAs, each ---------------------------------------
// A CTA walks its part of the row once, 16 logits per thread at a time, with
// running statistics per thread; the parts' statistics meet in the cluster's
// first CTA over distributed shared memory, so one launch serves one row as well
// as many and no workspace is shared between calls.
//
// The alternatives cost the walk nothing: each thread only knows its maximum
// and the batch it came from.  Call a thread's logits a unit, and its best (value,
// then lower index) the unit's key.  Whatever the K best logits of the part are,
// each is at least as good as the K-th best unit key, so they all stand in the
// K units with the best keys: these are read again (from L2: K / 256 of the
// part), what is at least as good as the K-th key is collected, and the K best of
// that are ranked by counting.
constexpr int LP_NT = 256;
constexpr int LP_CAND = 512;

// A part of a row as 16-byte vectors: vector j holds the logits 4 j - a ..
// 4 j - a + 3 of the part, a = how far the part starts past a 16-byte boundary.
struct LpPart {
  const float* base;  // the boundary at or below the part's first logit
  int a, end;         // its logits are base[a .. end)
  int64_t lo;         // the row index of base[0] (negative below the row's start)
  __device__ LpPart(const float* xr, int64_t lo_, int64_t hi) {
    const float* p = xr + lo_;
    a = (int)(((uintptr_t)p >> 2) & 3);
    base = p - a;
    end = a + (int)(hi > lo_ ? hi - lo_ : 0);
    lo = lo_ - a;
  }
  __device__ __forceinline__ float4 edge(int j) const {
    const int u = 4 * j;
    float4 v;
    v.x = u >= a && u < end ? base[u] : -INFINITY;
    v.y = u + 1 >= a && u + 1 < end ? base[u + 1] : -INFINITY;
    v.z = u + 2 >= a && u + 2 < end ? base[u + 2] : -INFINITY;
    v.w = u + 3 >= a && u + 3 < end ? base[u + 3] : -INFINITY;
    return v;
  }
  __device__ __forceinline__ float4 vec(int j) const {
    return 4 * j >= a && 4 * j + 4 <= end ? *reinterpret_cast<const float4*>(base + 4 * j) : edge(j);
  }
  // the 4 vectors of thread t in batch b
  __device__ __forceinline__ void batch(int b, int t, float4 (&v)[4]) const {
    const int j = b * 4 * LP_NT + t;
    if ((b > 0 || a == 0) && 4 * (b + 1) * 4 * LP_NT <= end) {
      const float4* p = reinterpret_cast<const float4*>(base) + j;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = p[q * LP_NT];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = vec(j + q * LP_NT);
    }
  }
};

struct LpShared {
  float f[8];
  LpStat part;                          // read by the cluster's first CTA
  unsigned long long top[LP_MAX_TOP];   // the part's alternatives, likewise
  unsigned long long unit[LP_NT];       // keys of the better units
  unsigned char owner[LP_NT];           // and their threads
  unsigned char chosen[LP_MAX_TOP];     // the threads of the K best
  unsigned long long cand[LP_CAND];
  unsigned long long k[8], least;
  int units, cands;
};

__device__ __forceinline__ float lp_block_max(float v, float* sh) {
  for (int o = 16; o > 0; o >>= 1) v = lp_max(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < LP_NT / 32; ++w) v = lp_max(v, sh[w]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float lp_block_sum(float v, float* sh) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < LP_NT / 32; ++w) v += sh[w];
  __syncthreads();
  return v;
}

// keys[0..n) into out[0..K) in order of rank (0 where there are fewer); keys differ
__device__ __forceinline__ void lp_rank(const unsigned long long* keys, int n, int K, unsigned long long* out) {
  if (threadIdx.x >= n && threadIdx.x < K) out[threadIdx.x] = 0ull;
  for (int i = threadIdx.x; i < n; i += LP_NT) {
    const unsigned long long k = keys[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += keys[j] > k;
    if (r < K) out[r] = k;
  }
}

// The K best keys of the part into sh.top.  m: this thread's maximum, mb: its batch.
__device__ void lp_select(const LpPart& p, float m, int mb, int K, LpShared& sh) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  // A value that at least K units reach: the least over the warps of each warp's
  // ceil(K / 8)-th largest maximum.
  float v = m;
  for (int size = 2; size <= 32; size <<= 1)
    for (int o = size >> 1; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, v, o);
      const bool down = (lane & size) == 0 || size == 32;  // larger values first
      v = ((lane & o) == 0) == down ? fmaxf(v, u) : fminf(v, u);
    }
  const int kq = (K + LP_NT / 32 - 1) / (LP_NT / 32);
  if (lane == kq - 1) sh.f[w] = v;
  if (t == 0) sh.units = sh.cands = 0;
  __syncthreads();
  float tau = sh.f[0];
#pragma unroll
  for (int i = 1; i < LP_NT / 32; ++i) tau = fminf(tau, sh.f[i]);
  if (m >= tau && m > -INFINITY) {  // where in its batch this unit's best stands
    float4 x[4];
    p.batch(mb, t, x);
    int at = 0;
#pragma unroll
    for (int q = 3; q >= 0; --q) {
      const int u = 4 * (mb * 4 * LP_NT + q * LP_NT + t);
      if (x[q].w == m) at = u + 3;
      if (x[q].z == m) at = u + 2;
      if (x[q].y == m) at = u + 1;
      if (x[q].x == m) at = u;
    }
    const int i = atomicAdd(&sh.units, 1);
    sh.unit[i] = lp_key(m, (uint32_t)(p.lo + at));
    sh.owner[i] = (unsigned char)t;
  }
  __syncthreads();
  const int n = sh.units, chosen = n < K ? n : K;
  if (t == 0 && n < K) sh.least = 0ull;
  if (t < n) {
    const unsigned long long k = sh.unit[t];
    int r = 0;
    for (int j = 0; j < n; ++j) r += sh.unit[j] > k;
    if (r < K) sh.chosen[r] = sh.owner[t];
    if (r == K - 1) sh.least = k;
  }
  __syncthreads();
  const unsigned long long least = sh.least;
  const int nv = (p.end + 3) >> 2;
  for (int s = w; s < chosen; s += LP_NT / 32)
    for (int j = sh.chosen[s] + LP_NT * lane; j < nv; j += LP_NT * 32) {
      const float4 q = p.vec(j);
      const float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const unsigned long long k = lp_key(e[c], (uint32_t)(p.lo + 4 * j + c));
        if (e[c] > -INFINITY && k >= least) {
          const int i = atomicAdd(&sh.cands, 1);
          if (i < LP_CAND) sh.cand[i] = k;
        }
      }
    }
  __syncthreads();
  const int nc = sh.cands;
  if (nc <= LP_CAND) {
    lp_rank(sh.cand, nc, K, sh.top);
    return;
  }
  // More than the list holds (a few units with most of the row's large values):
  // one alternative after the other, the best that is worse than the one before.
  unsigned long long last = ~0ull;
  for (int q = 0; q < K; ++q) {
    unsigned long long best = 0ull;
    for (int s = w; s < chosen; s += LP_NT / 32)
      for (int j = sh.chosen[s] + LP_NT * lane; j < nv; j += LP_NT * 32) {
        const float4 x = p.vec(j);
        const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const unsigned long long k = lp_key(e[c], (uint32_t)(p.lo + 4 * j + c));
          if (e[c] > -INFINITY && k < last && k > best) best = k;
        }
      }
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long u = __shfl_xor_sync(0xffffffffu, best, o);
      best = u > best ? u : best;
    }
    if (lane == 0) sh.k[w] = best;
    __syncthreads();
    for (int i = 0; i < LP_NT / 32; ++i) best = sh.k[i] > best ? sh.k[i] : best;
    if (t == 0) sh.top[q] = best;
    last = best;
    __syncthreads();
  }
}

__device__ __forceinline__ uint32_t lp_peer(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void lp_cluster_sync() {
  asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
}
__device__ __forceinline__ float lp_peer_f32(uint32_t at) {
  float f;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(at) : "memory");
  return f;
}
__device__ __forceinline__ unsigned long long lp_peer_u64(uint32_t at) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}

// parts: CTAs per row, the cluster's size
template <bool TOP>
__global__ void __launch_bounds__(LP_NT) k_logprobs_long(const float* __restrict__ x, int64_t ld,
                                                         const void* __restrict__ ids, int kind, int64_t V, int parts,
                                                         int K, float* __restrict__ logp, float* __restrict__ entropy,
                                                         float* __restrict__ stats, int32_t* __restrict__ top_ids,
                                                         float* __restrict__ top_logp) {
  ::tp::pdl_enter();
  __shared__ LpShared sh;
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - row * parts);
  const float* __restrict__ xr = x + row * ld;
  int tok = -1;
  float xt = 0.0f;
  if (part == 0 && t == 0 && logp) {
    tok = token_id(ids, kind, row);
    if (tok >= 0 && tok < V) xt = xr[tok];
  }
  const int64_t per = (V + parts - 1) / parts;
  const int64_t lo = per * part < V ? per * part : V, hi = lo + per < V ? lo + per : V;
  const LpPart p(xr, lo, hi);
  const int batches = (p.end + 16 * LP_NT - 1) / (16 * LP_NT);
  LpStat s{-INFINITY, 0.0f, 0.0f};
  int mb = 0;
  float4 next[4];
  p.batch(0, t, next);
  for (int b = 0; b < batches; ++b) {
    float4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = next[q];
    if (b + 1 < batches) p.batch(b + 1, t, next);
    float m = s.m;
#pragma unroll
    for (int q = 0; q < 4; ++q) m = lp_max(m, lp_max(lp_max(v[q].x, v[q].y), lp_max(v[q].z, v[q].w)));
    if (m != s.m) {
      s.move(m);
      mb = b;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s.add(v[q].x);
      s.add(v[q].y);
      s.add(v[q].z);
      s.add(v[q].w);
    }
  }
  const float own = s.m;
  s.move(lp_block_max(own, sh.f));
  s.S = lp_block_sum(s.S, sh.f);
  s.T = lp_block_sum(s.T, sh.f);
  if (TOP) {
    if (s.m < INFINITY) lp_select(p, own, mb, K, sh);  // not with a NaN or +inf in the part
    __syncthreads();
  }
  if (parts > 1) {
    if (t == 0) sh.part = s;
    lp_cluster_sync();
    if (part == 0) {
      float m = s.m;
      for (int c = 1; c < parts; ++c) m = lp_max(m, lp_peer_f32(lp_peer(&sh.part.m, c)));
      LpStat all{s.m, s.S, s.T};
      all.move(m);
      for (int c = 1; c < parts; ++c) {
        LpStat o{lp_peer_f32(lp_peer(&sh.part.m, c)), lp_peer_f32(lp_peer(&sh.part.S, c)),
                 lp_peer_f32(lp_peer(&sh.part.T, c))};
        o.move(m);
        all.S += o.S;
        all.T += o.T;
      }
      s = all;
      if (TOP && m < INFINITY) {
        // the parts' lists (0-padded) side by side, then the best of them
        const int n = parts * K;
        for (int i = t; i < n; i += LP_NT) {
          const int c = i / K;
          sh.cand[i] = lp_peer_u64(lp_peer(&sh.top[i - c * K], c));
        }
        __syncthreads();
        if (t < K) sh.top[t] = 0ull;
        __syncthreads();
        for (int i = t; i < n; i += LP_NT) {
          const unsigned long long k = sh.cand[i];
          int r = 0;
          for (int j = 0; j < n; ++j) r += sh.cand[j] > k;
          if (r < K && k) sh.top[r] = k;
        }
        __syncthreads();
      }
    }
    lp_cluster_sync();
    if (part != 0) return;
  }
  const LpRow r(s);
  if (t == 0) r.write(s, row, V, tok, xt, logp, entropy, stats);
  if (TOP && t < K) r.write_top(r.bad || r.none ? 0ull : sh.top[t], row * K + t, top_ids, top_logp);
}

// ---- gradient -------------------------------------------------------------------------
// What one row's values need: coefficients, statistics; zero: the row is zeros.
struct LpGrad {
  float m, lnS, c1, c2, H;
  int t;
  bool zero;
  __device__ LpGrad(int64_t row, int64_t V, const void* ids, int kind, const float* stats, const float* entropy,
                    const float* dlogp, const float* dentropy) {
    t = ids ? token_id(ids, kind, row) : -1;
    c1 = dlogp && t >= 0 ? dlogp[row] : 0.0f;
    c2 = dentropy ? dentropy[row] : 0.0f;
    m = stats[2 * row];
    lnS = stats[2 * row + 1];
    H = dentropy ? entropy[row] : 0.0f;
    zero = m == -INFINITY || (c1 == 0.0f && c2 == 0.0f);
    if (c2 == 0.0f) H = 0.0f;
    if (isnan(m) || (c1 != 0.0f && t >= V)) c1 = NAN;
  }
  __device__ __forceinline__ float operator()(float x, int64_t i) const {
    const float lp = fmaxf((x - m) - lnS, LP_FLOOR), p = lp_exp(lp);
    return c1 * ((i == t ? 1.0f : 0.0f) - p) - c2 * (p * (lp + H));
  }
};

// Rows of at most 1024 logits: a warp each.
__global__ void __launch_bounds__(256) k_logprobs_bwd_warp(const float* x, int64_t ld, const void* __restrict__ ids,
                                                           int kind, const float* __restrict__ stats,
                                                           const float* __restrict__ entropy,
                                                           const float* __restrict__ dlogp,
                                                           const float* __restrict__ dentropy, int64_t R, int V,
                                                           float* dx, int64_t ldd) {
  ::tp::pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= R) return;
  const float* xr = x + row * ld;
  float* dr = dx + row * ldd;
  const LpGrad g(row, V, ids, kind, stats, entropy, dlogp, dentropy);
  if (g.zero) {
    for (int i = lane; i < V; i += 32) dr[i] = 0.0f;
    return;
  }
  for (int i = lane; i < V; i += 256) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + 32 * k < V) v[k] = xr[i + 32 * k];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + 32 * k < V) dr[i + 32 * k] = g(v[k], i + 32 * k);
  }
}

// Longer rows: a CTA per 4096 logits, in 16-byte vectors where the row of x and
// the row of dx start at the same offset from a 16-byte boundary.
__global__ void __launch_bounds__(256) k_logprobs_bwd(const float* x, int64_t ld, const void* __restrict__ ids,
                                                      int kind, const float* __restrict__ stats,
                                                      const float* __restrict__ entropy,
                                                      const float* __restrict__ dlogp,
                                                      const float* __restrict__ dentropy, int64_t V, int chunks,
                                                      float* dx, int64_t ldd) {
  ::tp::pdl_enter();
  const int64_t row = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x - row * chunks);
  const float* xr = x + row * ld;
  float* dr = dx + row * ldd;
  const int a = (int)(((uintptr_t)xr >> 2) & 3);
  const LpGrad g(row, V, ids, kind, stats, entropy, dlogp, dentropy);
  if ((((uintptr_t)dr >> 2) & 3) == a) {
    const int end = a + (int)V;  // the row is base[a .. end)
    const float* xb = xr - a;
    float* db = dr - a;
    float4 v[4];
    int u[4];
    bool whole[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      u[q] = 4 * (chunk * 1024 + q * 256 + threadIdx.x);
      whole[q] = u[q] >= a && u[q] + 4 <= end;
      if (whole[q] && !g.zero) v[q] = *reinterpret_cast<const float4*>(xb + u[q]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = u[q] - a;
      if (whole[q]) {
        *reinterpret_cast<float4*>(db + u[q]) =
            g.zero ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                   : make_float4(g(v[q].x, i), g(v[q].y, i + 1), g(v[q].z, i + 2), g(v[q].w, i + 3));
      } else {
        for (int c = 0; c < 4; ++c)
          if (u[q] + c >= a && u[q] + c < end) db[u[q] + c] = g.zero ? 0.0f : g(xb[u[q] + c], i + c);
      }
    }
  } else {
    float v[16];
    const int64_t i0 = (int64_t)chunk * 4096 + threadIdx.x;
#pragma unroll
    for (int q = 0; q < 16; ++q)
      if (i0 + 256 * q < V && !g.zero) v[q] = xr[i0 + 256 * q];
#pragma unroll
    for (int q = 0; q < 16; ++q)
      if (i0 + 256 * q < V) dr[i0 + 256 * q] = g.zero ? 0.0f : g(v[q], i0 + 256 * q);
  }
}

// Rows up to this long are a warp's.
constexpr int64_t LP_WARP_MAX = 1024;

template <bool TOP>
static void launch_logprobs_warp(const float* x, int64_t ld, const void* ids, int kind, int64_t R, int V, int K,
                                 float* logp, float* entropy, float* stats, int32_t* top_ids, float* top_logp) {
  // one row per warp until there are warps for every scheduler several times over
  int per = 1;
  while (per < LP_ROWS && R >= (int64_t)sm_count() * 64 * 2 * per) per *= 2;
  const unsigned grid = (unsigned)((R + 8 * per - 1) / (8 * per));
#define TP_LP_WARP(N)                                                                                                 \
  if (V <= 32 * N) {                                                                                                  \
    TP_LAUNCH((k_logprobs_warp<N, TOP>), grid, 256, 0, x, ld, ids, kind, R, V, per, K, logp, entropy, stats, top_ids, \
              top_logp);                                                                                              \
    return;                                                                                                           \
  }
  TP_LP_WARP(1)
  TP_LP_WARP(2)
  TP_LP_WARP(3)
  TP_LP_WARP(4)
  TP_LP_WARP(6)
  TP_LP_WARP(8)
  TP_LP_WARP(9)
  TP_LP_WARP(12)
  TP_LP_WARP(16)
  TP_LP_WARP(20)
  TP_LP_WARP(24)
  TP_LP_WARP(28)
  TP_LP_WARP(32)
#undef TP_LP_WARP
}

// As TP_LAUNCH, in clusters of `cluster` CTAs.
template <typename... KArgs, typename... Args>
static void launch_cluster(void (*kernel)(KArgs...), unsigned grid, unsigned block, unsigned cluster, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.stream = stream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_pdl ? 2 : 1;
  TP_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
  g_launches++;
}

void launch_logprobs(const float* x, int64_t ld, const void* ids, int kind, int64_t R, int64_t V, int K, float* logp,
                     float* entropy, float* stats, int32_t* top_ids, float* top_logp) {
  if (R == 0) return;
  if (V <= LP_WARP_MAX) {
    if (K) launch_logprobs_warp<true>(x, ld, ids, kind, R, (int)V, K, logp, entropy, stats, top_ids, top_logp);
    else launch_logprobs_warp<false>(x, ld, ids, kind, R, (int)V, K, logp, entropy, stats, top_ids, top_logp);
    return;
  }
  // more CTAs per row while the rows alone leave SMs empty and a part keeps a batch
  int parts = 1;
  while (parts < 8 && R * parts < 4 * (int64_t)sm_count() && V / (2 * parts) >= 2048) parts *= 2;
  TP_REQUIRE(R * parts <= INT_MAX, "token_logprobs: %lld rows are too many", (long long)R);
  const unsigned grid = (unsigned)(R * parts);
  if (K)
    launch_cluster(k_logprobs_long<true>, grid, LP_NT, parts, x, ld, ids, kind, V, parts, K, logp, entropy, stats,
                   top_ids, top_logp);
  else
    launch_cluster(k_logprobs_long<false>, grid, LP_NT, parts, x, ld, ids, kind, V, parts, K, logp, entropy, stats,
                   top_ids, top_logp);
}

void launch_logprobs_bwd(const float* x, int64_t ld, const void* ids, int kind, const float* stats,
                         const float* entropy, const float* dlogp, const float* dentropy, int64_t R, int64_t V,
                         float* dx, int64_t ldd) {
  if (R == 0) return;
  if (V <= LP_WARP_MAX) {
    TP_LAUNCH(k_logprobs_bwd_warp, (unsigned)((R + 7) / 8), 256, 0, x, ld, ids, kind, stats, entropy, dlogp, dentropy,
              R, (int)V, dx, ldd);
    return;
  }
  const int chunks = (int)((V + 3 + 4095) / 4096);  // a row may start 3 logits past a boundary
  TP_REQUIRE(R * chunks <= INT_MAX, "token_logprobs_backward: %lld rows of %lld logits are too many", (long long)R,
             (long long)V);
  TP_LAUNCH(k_logprobs_bwd, (unsigned)(R * chunks), 256, 0, x, ld, ids, kind, stats, entropy, dlogp, dentropy, V,
            chunks, dx, ldd);
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
