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
//
// What bounds it: the logits' bytes.  Per logit there are about 7 issue slots (a
// difference, a clamp, a product, an exponential, two sums, a maximum), one of
// them a MUFU, of the 21 slots and 2.8 MUFU that an SM has in the time HBM takes
// to bring it.  8192 x 131072: 588 us, 7.3 TB/s read.
#include <cuda_runtime.h>

#include <cfloat>
#include <climits>

#include "tp_core.h"
#include "tp_launch.h"
#include "tp_token.cuh"

namespace tp {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_MAX_PARTS = 8;  // CTAs of a cluster

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

// Halves [lo, hi] towards the largest value that at least K of u[0..4) of the lanes
// of a group of L reach (as many reach lo).  For K near L: the K-th largest of L
// maxima lets L log(L / (L - K)) logits through, 112 of them for 32 of 32; of 4 L
// maxima it is 37.  (28014 x 1976 with 32 alternatives: 70.6 us, 303 without; with
// 20 62.1 and 63.8; with 11, of 32, 58.5 and 56.4, so from K = L / 2 on.)
template <int L>
__device__ __forceinline__ float lp_raise(const float (&u)[4], float lo, float hi, int K) {
  const unsigned group = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1) << (threadIdx.x & (32 - L));
  hi = fmaxf(hi, lo);  // -inf where nothing is left: lo stays above it
#pragma unroll 1
  for (int i = 0; i < 6; ++i) {
    const float mid = 0.5f * lo + 0.5f * hi;
    int n = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) n += __popc(__ballot_sync(0xffffffffu, u[q] >= mid) & group);
    if (n >= K) lo = mid;
    else hi = mid;
  }
  return lo;
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
};

// A thread's running statistics, 16 logits at a time.  Once the maximum's 1 is in
// S, a term below half a step of it, 2^-24, would be lost, and with it the thread's
// share of a tail that far down.  So 16 exponentials are summed among themselves,
// and what their sum loses on its way into S goes into the next one (Kahan's
// compensation): two roundings, however long the row is.  The maximum adds 0 to T,
// whose 16 terms are summed among themselves too.  (8192 x 131072: 588 us, one by
// one 585; 1999 x 50021 with 5 alternatives: 71.5, 70.6.)
struct LpRun : LpStat {
  float lost;  // of S
  __device__ __forceinline__ void move(float M) {
    lost *= lp_exp(fmaxf(m - M, LP_FLOOR));
    LpStat::move(M);
  }
  __device__ __forceinline__ void add(const float4 (&v)[4]) {
    float s[4], t[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float y0 = fmaxf(v[q].x - m, LP_FLOOR), y1 = fmaxf(v[q].y - m, LP_FLOOR);
      const float y2 = fmaxf(v[q].z - m, LP_FLOOR), y3 = fmaxf(v[q].w - m, LP_FLOOR);
      const float e0 = lp_exp(y0), e1 = lp_exp(y1), e2 = lp_exp(y2), e3 = lp_exp(y3);
      s[q] = (e0 + e1) + (e2 + e3);
      t[q] = fmaf(e3, y3, fmaf(e2, y2, fmaf(e1, y1, e0 * y0)));
    }
    const float more = ((s[0] + s[1]) + (s[2] + s[3])) - lost, sum = S + more;
    lost = (sum - S) - more;
    S = sum;
    T += (t[0] + t[1]) + (t[2] + t[3]);
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

// ---- short rows: a group of L lanes each, the row in registers --------------------------
// The row is read in 16-byte vectors from the boundary at or below its start:
// lane l of the group holds the vectors l + L k, k < N.  Smaller groups spend
// fewer instructions per row on exchanging (a warp works on 32 / L rows at
// once), larger ones finish a single row sooner.  The alternatives (K <= L of
// them): at least K logits are as large as the K-th largest of the lanes' maxima;
// what is that large is collected and the K best of it are ranked by counting.
// Where more is equal than the list holds, they are found one after the other.
// 65536 x 258: 12.9 us without alternatives (10.5 at HBM's rate), 19.8 with three:
// what picks them out of the registers is then as long as the rest.
template <int L, int N, bool TOP>
__global__ void __launch_bounds__(128) k_logprobs_short(const float* __restrict__ x, int64_t ld,
                                                        const void* __restrict__ ids, int kind, int64_t R, int V,
                                                        int K, float* __restrict__ logp, float* __restrict__ entropy,
                                                        float* __restrict__ stats, int32_t* __restrict__ top_ids,
                                                        float* __restrict__ top_logp) {
  ::tp::pdl_enter();
  constexpr unsigned ALL = 0xffffffffu;
  constexpr int G = 128 / L, CAND = 8 * L;
  __shared__ unsigned long long cand[TOP ? G : 1][TOP ? CAND : 1];
  __shared__ int cands[G];
  const int l = threadIdx.x % L, g = threadIdx.x / L;
  const int64_t row = (int64_t)blockIdx.x * G + g;
  const bool live = row < R;  // lanes without a row only take part in the exchanges
  const float* __restrict__ xr = x + row * ld;
  int t = -1;
  if (logp && live && l == 0) t = token_id(ids, kind, row);
  const int a = (int)(((uintptr_t)xr >> 2) & 3), end = live ? a + V : 0;  // the row is base[a .. end)
  const float* __restrict__ base = xr - a;
  float v[4 * N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int u = 4 * (l + L * k);
    if (u + 4 <= end && (k > 0 || u >= a)) {
      const float4 q = *reinterpret_cast<const float4*>(base + u);
      v[4 * k] = q.x, v[4 * k + 1] = q.y, v[4 * k + 2] = q.z, v[4 * k + 3] = q.w;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[4 * k + c] = u + c >= a && u + c < end ? base[u + c] : -INFINITY;
    }
  }
  const float xt = t >= 0 && t < V ? xr[t] : 0.0f;
  LpStat s{-INFINITY, 0.0f, 0.0f};
  float most[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int k = 4; k < 4 * N; ++k) most[k & 3] = lp_max(most[k & 3], v[k]);
  s.m = lp_max(lp_max(most[0], most[1]), lp_max(most[2], most[3]));
  float tau = s.m;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) s.m = lp_max(s.m, __shfl_xor_sync(ALL, s.m, o));
  float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of S: see LpRun
#pragma unroll
  for (int k = 0; k < 4 * N; ++k) {
    const float y = fmaxf(v[k] - s.m, LP_FLOOR), e = lp_exp(y);
    part[k & 3] += e;
    s.T = fmaf(e, y, s.T);
  }
  s.S = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    s.S += __shfl_xor_sync(ALL, s.S, o);
    s.T += __shfl_xor_sync(ALL, s.T, o);
  }
  const LpRow r(s);
  if (live && l == 0) r.write(s, row, V, t, xt, logp, entropy, stats);
  if constexpr (TOP) {
    auto index = [&](int k) { return 4 * (l + L * (k >> 2)) + (k & 3) - a; };  // of v[k] in the row
#pragma unroll
    for (int size = 2; size <= L; size <<= 1)  // the lanes' maxima in order, larger first
#pragma unroll
      for (int o = size >> 1; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(ALL, tau, o);
        tau = ((l & o) == 0) == ((l & size) == 0 || size == L) ? fmaxf(tau, u) : fminf(tau, u);
      }
    tau = fmaxf(__shfl_sync(ALL, tau, K - 1, L), -FLT_MAX);  // masked logits are no alternatives
    if (L > 8 && 2 * K > L) tau = lp_raise<L>(most, tau, s.m, K);
    unsigned long long some = 0ull;
    if (!r.bad) {
#pragma unroll
      for (int k = 0; k < 4 * N; ++k) some |= v[k] >= tau ? 1ull << k : 0ull;
    }
    if (l == 0) cands[g] = 0;
    __syncwarp();
    while (some) {
      const int i = index(__ffsll((long long)some) - 1), to = atomicAdd(&cands[g], 1);
      some &= some - 1;
      if (to < CAND) cand[g][to] = lp_key(xr[i], (uint32_t)i);
    }
    __syncwarp();
    const int n = cands[g];
    if (__any_sync(ALL, n > CAND)) {  // of any row of the warp
      unsigned long long last = ~0ull;
      for (int q = 0; q < K; ++q) {
        unsigned long long best = 0ull;
        for (int i = l; live && i < V; i += L) {  // from L1 or L2: registers for this would cost every row
          const unsigned long long y = lp_key(xr[i], (uint32_t)i);
          if (xr[i] > -INFINITY && y < last && y > best) best = y;
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) {
          const unsigned long long u = __shfl_xor_sync(ALL, best, o);
          best = u > best ? u : best;
        }
        last = best;
        if (live && l == 0) r.write_top(best, row * K + q, top_ids, top_logp);
      }
      return;
    }
    if (!live) return;
    if (l >= n && l < K) r.write_top(0ull, row * K + l, top_ids, top_logp);
    for (int i = l; i < n; i += L) {
      const unsigned long long y = cand[g][i];
      int above = 0;
      for (int j = 0; j < n; ++j) above += cand[g][j] > y;
      if (above < K) r.write_top(y, row * K + above, top_ids, top_logp);
    }
  }
}

// ---- longer rows: a team each -- a warp, a CTA or a cluster of CTAs ------------------------
// A team walks its part of the row once, 16 logits per thread at a time, with
// running statistics per thread.  Rows of a few thousand logits are a warp's: a
// CTA's barriers would cost them as much as the walk.  Where there are few rows, a
// cluster's CTAs take a part of one each; the parts' statistics meet in the
// cluster's first CTA over distributed shared memory, so one launch serves one
// row as well as many and no workspace is shared between calls.  (One row of
// 32000 with 20 alternatives: 7.0 us in eight parts, 36 us by a warp.  2000 rows of
// 50021 in two parts each: 95 us against 73, the exchange costs more than it
// balances.)  1999 x 50021 with 5 alternatives: 71 us, 5.6 TB/s: the last, uneven
// wave of rows is most of what is missing.
//
// The alternatives cost the walk little: of the q-th vectors of all its batches (a
// unit), each thread knows the largest maximum, where it stands and the largest of
// the others.  With tau a value that at least K units reach, the K best logits all
// stand in units that reach it.  Of such a unit one vector is read again, or all
// where another of its vectors reaches tau too (the row has mostly left L2 by
// then, so it matters how little that is); what reaches tau is collected, and the
// K best of it are ranked by counting.  Where so many logits are equal that a list
// overflows, whole threads are told apart by the index of their maximum too, which
// leaves exactly K of them.

// A part of a row as 16-byte vectors: vector j holds the logits 4 j - a ..
// 4 j - a + 3 of the part, a = how far the part starts past a 16-byte boundary.
// Batch b of thread t: the vectors 4 NT b + NT q + t, q < 4.
template <int NT>
struct LpPart {
  const float* base;  // the boundary at or below the part's first logit
  int a, end;         // its logits are base[a .. end)
  int64_t lo;         // the row index of base[0] (negative below the row's start)
  LpPart() = default;
  __device__ LpPart(const float* xr, int64_t lo_, int64_t hi) {
    const float* p = xr + lo_;
    a = (int)(((uintptr_t)p >> 2) & 3);
    base = p - a;
    end = a + (int)(hi > lo_ ? hi - lo_ : 0);
    lo = lo_ - a;
  }
  __device__ __forceinline__ int batches() const { return (end + 16 * NT - 1) / (16 * NT); }
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
  __device__ __forceinline__ void batch(int b, int t, float4 (&v)[4]) const {
    const int j = b * 4 * NT + t;
    if ((b > 0 || a == 0) && 16 * NT * (b + 1) <= end) {
      const float4* p = reinterpret_cast<const float4*>(base) + j;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = p[q * NT];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = vec(j + q * NT);
    }
  }
};

template <int NT>
struct LpShared {
  static constexpr int CAND = NT == 32 ? 256 : 512;  // collected logits
  static constexpr int LIST = NT == 32 ? 128 : 256;  // vectors, and units, read again
  LpStat warp[NT / 32];
  float kth[NT / 32];                  // per warp: a value that K / (NT / 32) of its threads' maxima reach
  unsigned long long top[LP_MAX_TOP];  // the part's alternatives
  int vector[LIST];                    // vectors read again
  unsigned short chosen[LIST];         // units read again whole: 4 thread + vector
  unsigned short owner[NT];            // ties: threads
  unsigned long long cand[CAND];
  unsigned long long k[NT / 32], least;
  int vectors, units, cands;
};

// Where the cluster's CTAs leave what their parts came to: in the first one.
struct LpGather {
  LpStat part[LP_MAX_PARTS];
  unsigned long long top[LP_MAX_PARTS * LP_MAX_TOP];
};

template <int NT>
__device__ __forceinline__ void lp_sync() {
  if (NT == 32) __syncwarp();
  else __syncthreads();
}

// the warp's largest value; a NaN in any lane is kept (which an unsigned maximum of
// order-preserving bits does not do: the compiler makes it a float one without)
__device__ __forceinline__ float lp_warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// the warp's values in order, larger first
__device__ __forceinline__ float lp_sorted(float v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, v, o);
      v = ((lane & o) == 0) == ((lane & size) == 0) ? fmaxf(v, u) : fminf(v, u);
    }
  return v;
}

// keys[0..n) into out[0..K) in order of rank (0 where there are fewer); keys differ
template <int NT>
__device__ __forceinline__ void lp_rank(int t, const unsigned long long* keys, int n, int K, unsigned long long* out) {
  if (t >= n && t < K) out[t] = 0ull;
  for (int i = t; i < n; i += NT) {
    const unsigned long long k = keys[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += keys[j] > k;
    if (r < K) out[r] = k;
  }
}

// Shows `take` every logit of the units chosen[0..n), by all threads of the team.
template <int NT, class F>
__device__ __forceinline__ void lp_reread(int t, const LpPart<NT>& p, const unsigned short* chosen, int n, F take) {
  const int nv = (p.end + 3) >> 2, per = p.batches();
  // i / per in f32: i < 2^21 and i / per < 256 are off by less than 2^-23 of
  // themselves, 3.1e-5; (i + 0.5) / per is 0.5 / per off a whole number, which at the
  // most batches there are, 8192 (2^24 logits by 128 threads), is 6.1e-5.
  const float inv = 1.0f / (float)per;
  for (int i0 = t; i0 < n * per; i0 += 2 * NT) {
    float4 q[2];
    int j[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int i = i0 + c * NT, s = (int)(((float)i + 0.5f) * inv);
      j[c] = nv;
      if (i < n * per) {
        const int code = chosen[s];
        j[c] = 4 * NT * (i - s * per) + NT * (code & 3) + (code >> 2);
      }
      if (j[c] < nv) q[c] = p.vec(j[c]);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (j[c] < nv) {
        const uint32_t at = (uint32_t)(p.lo + 4 * j[c]);
        take(q[c].x, at);
        take(q[c].y, at + 1);
        take(q[c].z, at + 2);
        take(q[c].w, at + 3);
      }
  }
}

template <int NT>
__device__ __forceinline__ void lp_add(LpShared<NT>& sh, float x, uint32_t at) {
  const int i = atomicAdd(&sh.cands, 1);
  if (i < LpShared<NT>::CAND) sh.cand[i] = lp_key(x, at);
}

// lp_select where ties overflow a list: threads in the place of units.  m: this
// thread's maximum if it is one of those that reach tau, else -inf.  Not inlined:
// what it needs in registers is not held through the walk.
template <int NT>
__device__ __noinline__ void lp_select_ties(int t, const float* base, int a, int end, int64_t lo, float m, int mb,
                                            int K, LpShared<NT>& sh) {
  LpPart<NT> p;
  p.base = base;
  p.a = a;
  p.end = end;
  p.lo = lo;
  lp_sync<NT>();
  if (t == 0) sh.units = sh.cands = 0, sh.least = 0ull;
  lp_sync<NT>();
  if (m > -INFINITY) {
    float4 x[4];
    p.batch(mb, t, x);
    int at = 0;
#pragma unroll
    for (int q = 3; q >= 0; --q) {
      const int u = 4 * (mb * 4 * NT + q * NT + t);
      if (x[q].w == m) at = u + 3;
      if (x[q].z == m) at = u + 2;
      if (x[q].y == m) at = u + 1;
      if (x[q].x == m) at = u;
    }
    const int i = atomicAdd(&sh.units, 1);
    sh.cand[i] = lp_key(m, (uint32_t)(p.lo + at));
    sh.owner[i] = (unsigned short)t;
  }
  lp_sync<NT>();
  const int n = sh.units;
  const int chosen = 4 * (n < K ? n : K);
  for (int u = t; u < n; u += NT) {
    const unsigned long long k = sh.cand[u];
    int above = 0;
    for (int j = 0; j < n; ++j) above += sh.cand[j] > k;
    if (above < K)
      for (int q = 0; q < 4; ++q) sh.chosen[4 * above + q] = (unsigned short)(4 * sh.owner[u] + q);
    if (above == K - 1) sh.least = k;
  }
  lp_sync<NT>();
  const unsigned long long least = sh.least;
  lp_reread<NT>(t, p, sh.chosen, chosen, [&](float x, uint32_t at) {
    if (x > -INFINITY && lp_key(x, at) >= least) lp_add(sh, x, at);
  });
  lp_sync<NT>();
  const int nc = sh.cands;
  if (nc <= LpShared<NT>::CAND) {
    lp_rank<NT>(t, sh.cand, nc, K, sh.top);
    return;
  }
  // More than the list holds (a few threads with most of the row's large values):
  // one alternative after the other, the best that is worse than the one before.
  unsigned long long last = ~0ull;
  for (int q = 0; q < K; ++q) {
    unsigned long long best = 0ull;
    lp_reread<NT>(t, p, sh.chosen, chosen, [&](float x, uint32_t at) {
      const unsigned long long k = lp_key(x, at);
      if (x > -INFINITY && k < last && k > best) best = k;
    });
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long u = __shfl_xor_sync(0xffffffffu, best, o);
      best = u > best ? u : best;
    }
    if ((t & 31) == 0) sh.k[t >> 5] = best;
    lp_sync<NT>();
    for (int i = 0; i < NT / 32; ++i) best = sh.k[i] > best ? sh.k[i] : best;
    if (t == 0) sh.top[q] = best;
    last = best;
    lp_sync<NT>();
  }
}

// What a thread knows of the q-th vectors of its batches: the largest maximum, the
// batch it came from first, and the largest of the others.
struct LpUnit {
  float m, next;
  int batch;
};

// The K best keys of the part into sh.top, by thread t of the team.  tau: a value
// that at least K units reach; the counters are 0.
template <int NT>
__device__ void lp_select(int t, const LpPart<NT>& p, const LpUnit (&unit)[4], float tau, int K, LpShared<NT>& sh) {
  tau = fmaxf(tau, -FLT_MAX);  // masked logits are no alternatives
  bool in = false;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (unit[q].m >= tau) {
      in = true;
      if (unit[q].next < tau) {
        const int i = atomicAdd(&sh.vectors, 1);
        if (i < LpShared<NT>::LIST) sh.vector[i] = 4 * NT * unit[q].batch + NT * q + t;
      } else {
        const int i = atomicAdd(&sh.units, 1);
        if (i < LpShared<NT>::LIST) sh.chosen[i] = (unsigned short)(4 * t + q);
      }
    }
  lp_sync<NT>();
  const int vectors = sh.vectors, units = sh.units;
  if (vectors <= LpShared<NT>::LIST && units <= LpShared<NT>::LIST) {
    auto take = [&](float x, uint32_t at) {
      if (x >= tau) lp_add(sh, x, at);
    };
    for (int i = t; i < vectors; i += NT) {
      const int j = sh.vector[i];
      const float4 x = p.vec(j);
      const uint32_t at = (uint32_t)(p.lo + 4 * j);
      take(x.x, at);
      take(x.y, at + 1);
      take(x.z, at + 2);
      take(x.w, at + 3);
    }
    if (units) lp_reread<NT>(t, p, sh.chosen, units, take);
    lp_sync<NT>();
    const int nc = sh.cands;
    if (nc <= LpShared<NT>::CAND) {
      lp_rank<NT>(t, sh.cand, nc, K, sh.top);
      return;
    }
  }
  // the thread's largest, and where it came from first
  float m = unit[0].m;
  int mb = unit[0].batch;
#pragma unroll
  for (int q = 1; q < 4; ++q)
    if (unit[q].m > m || (unit[q].m == m && unit[q].batch < mb)) m = unit[q].m, mb = unit[q].batch;
  lp_select_ties<NT>(t, p.base, p.a, p.end, p.lo, in ? m : -INFINITY, mb, K, sh);
}

// p's place in the cluster's first CTA
__device__ __forceinline__ uint32_t lp_first(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)));
  return r;
}
__device__ __forceinline__ void lp_put(uint32_t at, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}
__device__ __forceinline__ void lp_put(uint32_t at, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}

// NT: threads of a team (a warp: four teams to a CTA); SPLIT: a row is a cluster's,
// of `parts` CTAs.  Few CTAs have the SMs to themselves then, so each fetches its
// next batch ahead (64 x 131072 with 20 alternatives: 16.5 us, 18.2 without; with every
// SM full the registers for it cost more than it brings, 619 us against 590 for
// 8192 x 131072).
template <int NT, bool TOP, bool SPLIT>
__global__ void __launch_bounds__(NT == 32 ? 128 : NT)
    k_logprobs_long(const float* __restrict__ x, int64_t ld, const void* __restrict__ ids, int kind, int64_t R,
                    int64_t V, int parts, int K, float* __restrict__ logp, float* __restrict__ entropy,
                    float* __restrict__ stats, int32_t* __restrict__ top_ids, float* __restrict__ top_logp) {
  ::tp::pdl_enter();
  constexpr int TEAMS = NT == 32 ? 4 : 1, WARPS = NT / 32;
  __shared__ LpShared<NT> shared[TEAMS];
  __shared__ LpGather all;
  // the first CTA has to be there before another writes to it: asked here, waited for below
  if (SPLIT) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  LpShared<NT>& sh = shared[threadIdx.x / NT];
  const int t = threadIdx.x % NT, lane = t & 31;
  int64_t row;
  int part = 0;
  if (NT == 32) {
    row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / NT;
    if (row >= R) return;
  } else if (SPLIT) {
    row = blockIdx.x / parts;
    part = (int)(blockIdx.x - row * parts);
  } else {
    row = blockIdx.x;
  }
  const float* __restrict__ xr = x + row * ld;
  int tok = -1;
  float xt = 0.0f;
  if (part == 0 && t == 0 && logp) {
    tok = token_id(ids, kind, row);
    if (tok >= 0 && tok < V) xt = xr[tok];
  }
  const int64_t per = SPLIT ? (V + parts - 1) / parts : V;
  const int64_t lo = per * part < V ? per * part : V, hi = lo + per < V ? lo + per : V;
  const LpPart<NT> p(xr, lo, hi);
  const int batches = p.batches();
  LpRun run;
  run.m = -INFINITY;
  run.S = run.T = run.lost = 0.0f;
  LpUnit unit[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) unit[q] = LpUnit{-INFINITY, -INFINITY, 0};
  float4 next[SPLIT ? 4 : 1];
  if constexpr (SPLIT) p.batch(0, t, next);
  for (int b = 0; b < batches; ++b) {
    float4 v[4];
    if constexpr (SPLIT) {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = next[q];
      if (b + 1 < batches) p.batch(b + 1, t, next);
    } else {
      p.batch(b, t, v);
    }
    float m;
    if (TOP) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float y = lp_max(lp_max(v[q].x, v[q].y), lp_max(v[q].z, v[q].w));
        unit[q].next = fmaxf(unit[q].next, fminf(unit[q].m, y));
        if (y > unit[q].m) unit[q].batch = b;
        unit[q].m = lp_max(unit[q].m, y);
      }
      m = lp_max(lp_max(unit[0].m, unit[1].m), lp_max(unit[2].m, unit[3].m));
    } else {
      m = run.m;
#pragma unroll
      for (int q = 0; q < 4; ++q) m = lp_max(m, lp_max(lp_max(v[q].x, v[q].y), lp_max(v[q].z, v[q].w)));
    }
    if (m != run.m) run.move(m);
    run.add(v);
  }
  LpStat s = run;
  float own = s.m;
  const float most = lp_warp_max(own);
  s.move(most);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.S += __shfl_xor_sync(0xffffffffu, s.S, o);
    s.T += __shfl_xor_sync(0xffffffffu, s.T, o);
  }
  float tau = most;
  if (TOP) {  // the ceil(K / WARPS)-th largest of the threads' maxima, equal ones counted once
    const int kq = (K + WARPS - 1) / WARPS;
    if (kq <= 5) {
      for (int i = 1; i < kq; ++i) {
        if (own == tau) own = -INFINITY;
        tau = lp_warp_max(own);
      }
    } else {
      tau = lp_sorted(own, lane);
      tau = __shfl_sync(0xffffffffu, tau, kq - 1);
    }
    if (NT == 32 && K > 16) {
      const float u[4] = {unit[0].m, unit[1].m, unit[2].m, unit[3].m};
      tau = lp_raise<32>(u, fmaxf(tau, -FLT_MAX), most, K);
    }
    if (t == 0) sh.vectors = sh.units = sh.cands = 0, sh.least = 0ull;
  }
  if (WARPS > 1) {
    if (lane == 0) {
      sh.warp[t >> 5] = s;
      sh.kth[t >> 5] = tau;
    }
    __syncthreads();
    s = sh.warp[0];
    float m = s.m;
#pragma unroll
    for (int i = 1; i < WARPS; ++i) m = lp_max(m, sh.warp[i].m);
    if (t < 32) {  // the sums are the first warp's business
      s.move(m);
#pragma unroll
      for (int i = 1; i < WARPS; ++i) {
        LpStat o = sh.warp[i];
        o.move(m);
        s.S += o.S;
        s.T += o.T;
      }
    }
    s.m = m;
    if (TOP) {
      tau = sh.kth[0];
#pragma unroll
      for (int i = 1; i < WARPS; ++i) tau = fminf(tau, sh.kth[i]);
    }
  }
  if (TOP) {
    if (WARPS == 1) __syncwarp();
    if (s.m < INFINITY) lp_select<NT>(t, p, unit, tau, K, sh);  // not with a NaN or +inf in the part
    lp_sync<NT>();
  }
  if (SPLIT) {
    asm volatile("barrier.cluster.wait;" ::: "memory");
    if (t == 0) {
      const uint32_t at = lp_first(&all.part[part]);
      lp_put(at, s.m);
      lp_put(at + 4, s.S);
      lp_put(at + 8, s.T);
    }
    if (TOP && t < K) lp_put(lp_first(&all.top[part * K + t]), sh.top[t]);
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    if (part != 0) return;
    s = all.part[0];
    float m = s.m;
    for (int c = 1; c < parts; ++c) m = lp_max(m, all.part[c].m);
    s.move(m);
    for (int c = 1; c < parts; ++c) {
      LpStat o = all.part[c];
      o.move(m);
      s.S += o.S;
      s.T += o.T;
    }
    if (TOP && m < INFINITY) {
      // the parts' lists (0-padded) side by side, then the best of them
      const int n = parts * K;
      if (t < K) sh.top[t] = 0ull;
      __syncthreads();
      if (t < n) {
        const unsigned long long k = all.top[t];
        int r = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) r += all.top[j] > k;
        if (r < K && k) sh.top[r] = k;
      }
      __syncthreads();
    }
  }
  if (t >= 32) return;
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

// Rows of at most 1024 logits: a group of L lanes each, in 16-byte vectors where
// the row of x and the row of dx start at the same offset from a boundary.
// 8 lanes have 32 vectors under way, 32 lanes 128 but four times as many CTAs and
// rows' coefficients: us by 8 / by 32 lanes,
//
//    rows      64          200         258         300         400         500
//    9500   5.1/ 5.2    5.2/ 5.1    6.7/ 5.7    6.2/ 5.3    7.8/ 6.7
//   15000   5.1/ 6.1    5.2/ 7.1    9.3/ 8.8    9.7/10.0   12.2/11.8
//   19000   5.1/ 7.2    7.3/ 9.6   11.0/12.9   11.0/12.8   13.6/14.3
//   65536   9.5/25.8   20.2/31.4   26.9/36.2   29.0/36.7   35.9/40.5   45.2/44.0 logits
// A row without an upstream gradient is read no further than its lanes' first 16
// values, which are fetched before that is known: 65536 x 1000, 90% ignored, 64.8
// us (49.4 if it were known first, but 81.8 instead of 79.9 with none ignored).
template <int L>
__global__ void __launch_bounds__(128) k_logprobs_bwd_short(const float* x, int64_t ld, const void* __restrict__ ids,
                                                            int kind, const float* __restrict__ stats,
                                                            const float* __restrict__ entropy,
                                                            const float* __restrict__ dlogp,
                                                            const float* __restrict__ dentropy, int64_t R, int V,
                                                            float* dx, int64_t ldd) {
  ::tp::pdl_enter();
  const int l = threadIdx.x % L;
  const int64_t row = (int64_t)blockIdx.x * (128 / L) + threadIdx.x / L;
  if (row >= R) return;
  const float* xr = x + row * ld;
  float* dr = dx + row * ldd;
  const int a = (int)(((uintptr_t)xr >> 2) & 3);
  if ((((uintptr_t)dr >> 2) & 3) == a) {
    const int end = a + V;  // the row is base[a .. end)
    const float* xb = xr - a;
    float* db = dr - a;
    float4 v[4];
    auto whole = [&](int u) { return u >= a && u + 4 <= end; };
    auto load = [&](int j) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (whole(4 * (j + L * q))) v[q] = *reinterpret_cast<const float4*>(xb + 4 * (j + L * q));
    };
    load(l);  // under way while the row's coefficients are fetched
    const LpGrad g(row, V, ids, kind, stats, entropy, dlogp, dentropy);
    for (int j = l; 4 * j < end; j += 4 * L) {
      if (j > l && !g.zero) load(j);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int u = 4 * (j + L * q), i = u - a;
        if (whole(u)) {
          *reinterpret_cast<float4*>(db + u) =
              g.zero ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                     : make_float4(g(v[q].x, i), g(v[q].y, i + 1), g(v[q].z, i + 2), g(v[q].w, i + 3));
        } else {
          for (int c = 0; c < 4; ++c)
            if (u + c >= a && u + c < end) db[u + c] = g.zero ? 0.0f : g(xb[u + c], i + c);
        }
      }
    }
  } else {
    const LpGrad g(row, V, ids, kind, stats, entropy, dlogp, dentropy);
    for (int i = l; i < V; i += 8 * L) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + L * k < V && !g.zero) v[k] = xr[i + L * k];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + L * k < V) dr[i + L * k] = g.zero ? 0.0f : g(v[k], i + L * k);
    }
  }
}

constexpr int LP_BWD_NT = 128;

// Longer rows: a CTA per 2048 logits, in 16-byte vectors where the row of x and
// the row of dx start at the same offset from a 16-byte boundary.  (32 registers,
// so that every thread an SM can hold has its 64 bytes of loads in flight: 4096 x
// 32000 takes 155 us, 178 with 43 registers.  CTAs of 256 threads: the same for
// long rows, 65536 x 1500 186 us instead of 134.)
__global__ void __launch_bounds__(LP_BWD_NT, 2048 / LP_BWD_NT) k_logprobs_bwd(const float* x, int64_t ld, const void* __restrict__ ids,
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
      u[q] = 4 * (chunk * 4 * LP_BWD_NT + q * LP_BWD_NT + (int)threadIdx.x);
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
    const int64_t i0 = (int64_t)chunk * 16 * LP_BWD_NT + threadIdx.x;
#pragma unroll
    for (int q = 0; q < 16; ++q)
      if (i0 + LP_BWD_NT * q < V && !g.zero) v[q] = xr[i0 + LP_BWD_NT * q];
#pragma unroll
    for (int q = 0; q < 16; ++q)
      if (i0 + LP_BWD_NT * q < V) dr[i0 + LP_BWD_NT * q] = g.zero ? 0.0f : g(v[q], i0 + LP_BWD_NT * q);
  }
}

// Rows up to this long are held in registers.
constexpr int64_t LP_SHORT = 1024;
// Rows up to this long are 8 lanes' in the gradient (in two rounds of loads), and
// up to this long if there are many (k_logprobs_bwd_short).
constexpr int64_t LP_BWD_8 = 253, LP_BWD_8_MANY = 400;

template <int L, bool TOP>
static void launch_logprobs_short(const float* x, int64_t ld, const void* ids, int kind, int64_t R, int V, int K,
                                  float* logp, float* entropy, float* stats, int32_t* top_ids, float* top_logp) {
  const unsigned grid = (unsigned)((R + 128 / L - 1) / (128 / L));
#define TP_LP_SHORT(N)                                                                                             \
  if (V + 3 <= 4 * L * N) { /* a row may start 3 logits past a boundary */                                         \
    TP_LAUNCH((k_logprobs_short<L, N, TOP>), grid, 128, 0, x, ld, ids, kind, R, V, K, logp, entropy, stats, top_ids, \
              top_logp);                                                                                           \
    return;                                                                                                        \
  }
  TP_LP_SHORT(1)
  TP_LP_SHORT(2)
  TP_LP_SHORT(3)
  TP_LP_SHORT(4)
  TP_LP_SHORT(5)
  TP_LP_SHORT(6)
  TP_LP_SHORT(7)
  TP_LP_SHORT(8)
  TP_LP_SHORT(9)
#undef TP_LP_SHORT
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

// Threads of a row's team.  Times in us, 512 MB of logits, without / with 5 / with
// 20 alternatives:
//
//          4096         8192          12000         16384         24000          50021 logits a row
//   warp   83/ 97/124   83/ 93/108    91/ 98/109    91/ 99/112    101/107/121    101/109/125
//   128   101/153/166   87/112/120    89/108/111    88/102/105     86/ 98/102     93/101/103
//   256   105/178/201   83/129/144    83/113/123    83/106/110     80/100/107     90/ 97/101
//
// A warp's row has no barrier; more threads have fewer batches each, which is worth
// more the fewer alternatives there are to pick.  1999 rows of 50021 with 5: 100, 70
// and 74 us (the last rows of a wave are less alone with 128); 64 rows of 4096 with
// 20: 9.4, 5.1 and 6.6.
static int lp_threads(int64_t R, int64_t V, int K) {
  const int64_t sms = sm_count();
  if (R >= 16 * sms) {
    if (V <= (K ? 12288 : 8192)) return 32;
    return K && V <= 24576 ? 128 : 256;
  }
  return V <= 4096 || R >= 6 * sms ? 128 : 256;
}

void launch_logprobs(const float* x, int64_t ld, const void* ids, int kind, int64_t R, int64_t V, int K, float* logp,
                     float* entropy, float* stats, int32_t* top_ids, float* top_logp) {
  if (R == 0) return;
  if (V <= LP_SHORT) {
    // the smallest group whose lanes hold the row and whose warps still fill the SMs
    const int64_t warps = (int64_t)sm_count() * 16;
    const int L = V <= 8 * 36 - 3 && K <= 8 && R >= 4 * warps ? 8
                  : (V <= 16 * 36 - 3 && K <= 16 && R >= 2 * warps ? 16 : 32);
#define TP_LP_GROUP(L)                                                                                                \
  if (K) launch_logprobs_short<L, true>(x, ld, ids, kind, R, (int)V, K, logp, entropy, stats, top_ids, top_logp);   \
  else launch_logprobs_short<L, false>(x, ld, ids, kind, R, (int)V, K, logp, entropy, stats, top_ids, top_logp);
    if (L == 8) {
      TP_LP_GROUP(8)
    } else if (L == 16) {
      TP_LP_GROUP(16)
    } else {
      TP_LP_GROUP(32)
    }
#undef TP_LP_GROUP
    return;
  }
  const int nt = lp_threads(R, V, K);
  // more CTAs per row while the rows alone leave SMs empty and a part keeps half a batch
  int parts = 1;
  while (nt == 256 && parts < LP_MAX_PARTS && R * parts < 4 * (int64_t)sm_count() && V / (2 * parts) >= 2048) parts *= 2;
  const int64_t ctas = nt == 32 ? (R + 3) / 4 : R * parts;
  TP_REQUIRE(ctas <= INT_MAX, "token_logprobs: %lld rows are too many", (long long)R);
#define TP_LP_LONG(NT, TOP, SPLIT)                                                                                  \
  launch_cluster(k_logprobs_long<NT, TOP, SPLIT>, (unsigned)ctas, NT == 32 ? 128 : NT, parts, x, ld, ids, kind, R, V, \
                 parts, K, logp, entropy, stats, top_ids, top_logp)
  if (nt == 32 && K) TP_LP_LONG(32, true, false);
  else if (nt == 32) TP_LP_LONG(32, false, false);
  else if (nt == 128 && K) TP_LP_LONG(128, true, false);
  else if (nt == 128) TP_LP_LONG(128, false, false);
  else if (parts > 1 && K) TP_LP_LONG(256, true, true);
  else if (parts > 1) TP_LP_LONG(256, false, true);
  else if (K) TP_LP_LONG(256, true, false);
  else TP_LP_LONG(256, false, false);
#undef TP_LP_LONG
}

void launch_logprobs_bwd(const float* x, int64_t ld, const void* ids, int kind, const float* stats,
                         const float* entropy, const float* dlogp, const float* dentropy, int64_t R, int64_t V,
                         float* dx, int64_t ldd) {
  if (R == 0) return;
  if (V <= LP_SHORT) {
#define TP_LP_BWD(L)                                                                                                 \
  TP_LAUNCH(k_logprobs_bwd_short<L>, (unsigned)((R + 128 / L - 1) / (128 / L)), 128, 0, x, ld, ids, kind, stats, entropy, \
            dlogp, dentropy, R, (int)V, dx, ldd)
    if (V <= LP_BWD_8 || (V <= LP_BWD_8_MANY && R >= (int64_t)sm_count() * 112)) TP_LP_BWD(8);
    else TP_LP_BWD(32);
#undef TP_LP_BWD
    return;
  }
  const int chunks = (int)((V + 3 + 16 * LP_BWD_NT - 1) / (16 * LP_BWD_NT));  // a row may start 3 logits past a boundary
  TP_REQUIRE(R * chunks <= INT_MAX, "token_logprobs_backward: %lld rows of %lld logits are too many", (long long)R,
             (long long)V);
  TP_LAUNCH(k_logprobs_bwd, (unsigned)(R * chunks), LP_BWD_NT, 0, x, ld, ids, kind, stats, entropy, dlogp, dentropy, V,
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
    check_aligned({logits, ids, logp, entropy, stats, top_ids, top_logp}, what);
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
    check_aligned({logits, ids, stats, entropy, dlogp, dentropy, dlogits}, what);
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
