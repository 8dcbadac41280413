// Fused optimizer steps: one multi-tensor launch per parameter group.
//
// Reference: adam_step.wgsl / adamw_step.wgsl / sgd_step.wgsl update one
// parameter per dispatch (three uniform buffers each, reductionOps.ts:533-653)
// and the Python optimizers loop over parameters (optim/__init__.py:158-205,
// 238-312, 345-418).  Here a device table lists every tensor of the group and a
// chunk table splits them into 64K-element chunks; a grid sized to the SM
// count walks the chunks with 128-bit loads, reading param, grad and state
// once and writing param and state once (AdamW: 28 B per element, SGD with
// momentum: 20 B).
//
// The per-element arithmetic is the WGSL's, operation by operation, with
// explicit round-to-nearest intrinsics so no multiply-add is contracted: the
// result is bit-identical to the CPU oracle's restatement compiled with
// -ffp-contract=off (sqrt and division are IEEE-rounded in both).
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <unordered_map>

#include "tp_core.h"
#include "tp_launch.h"
#include "tp_token.cuh"

namespace tp {

constexpr int64_t OPT_CHUNK = 65536;

struct OptRow {
  float* p;
  const float* g;
  float* s0;
  float* s1;
  float* lo;  // SGD: the updated parameter's tf32 low parts (optional)
  int64_t n;
};
struct OptChunk {
  int32_t row;
  int32_t len;
  int64_t start;
};

struct AdamHP {
  float lr, b1, b2, eps, wd, step_size, inv_sqrt_bc2, omb1, omb2, lrwd;
};

// Narrows a chunk to the part that item `c` stands for (chunk c >> part_log);
// false: there is none.
__device__ __forceinline__ bool opt_part(OptChunk& ch, int c, int part_log) {
  const int len = (int)(OPT_CHUNK >> part_log), from = (c & ((1 << part_log) - 1)) * len;
  if (from >= ch.len) return false;
  ch.start += from;
  ch.len = ch.len - from < len ? ch.len - from : len;
  return true;
}

// adamw_step.wgsl:26-39 (ADAMW) and adam_step.wgsl:25-38 (ADAM).
template <bool ADAMW>
__device__ __forceinline__ void adam_elem(float& p, float g, float& m, float& v, const AdamHP& h) {
  if (ADAMW) {
    if (h.wd != 0.0f) p = __fsub_rn(p, __fmul_rn(h.lrwd, p));
  } else {
    if (h.wd != 0.0f) g = __fadd_rn(g, __fmul_rn(h.wd, p));
  }
  m = __fadd_rn(__fmul_rn(m, h.b1), __fmul_rn(h.omb1, g));
  v = __fadd_rn(__fmul_rn(v, h.b2), __fmul_rn(__fmul_rn(h.omb2, g), g));
  float denom = __fadd_rn(__fmul_rn(__fsqrt_rn(v), h.inv_sqrt_bc2), h.eps);
  float upd = __fmul_rn(__fdiv_rn(m, denom), h.step_size);
  p = __fsub_rn(p, upd);
}

// SCALED: each gradient is multiplied by *gs on read (rounded once, as a pass
// that scales the gradients in place rounds it), and a CTA takes 1 / 2^part_log
// of a chunk at a time: 2.3 M parameters in 45 chunks take 53 us whole, 18.6 in
// 32 parts.
template <bool ADAMW, bool SCALED>
__global__ void __launch_bounds__(256) k_adam_multi(const OptRow* __restrict__ rows, const OptChunk* __restrict__ chunks,
                                                    int nchunks, AdamHP h, const float* __restrict__ gs,
                                                    int part_log) {
  ::tp::pdl_enter();
  const float s = SCALED ? *gs : 1.0f;
  if (!SCALED) part_log = 0;
  auto scaled = [&](float4 g) {
    return SCALED ? make_float4(__fmul_rn(g.x, s), __fmul_rn(g.y, s), __fmul_rn(g.z, s), __fmul_rn(g.w, s)) : g;
  };
  for (int c = blockIdx.x; c < nchunks << part_log; c += gridDim.x) {
    OptChunk ch = chunks[c >> part_log];
    if (SCALED && !opt_part(ch, c, part_log)) continue;
    OptRow r = rows[ch.row];
    float* __restrict__ P = r.p + ch.start;
    const float* __restrict__ G = r.g + ch.start;
    float* __restrict__ M = r.s0 + ch.start;
    float* __restrict__ V = r.s1 + ch.start;
    int len = ch.len;
    int len4 = len >> 2;
    float4* P4 = reinterpret_cast<float4*>(P);
    const float4* G4 = reinterpret_cast<const float4*>(G);
    float4* M4 = reinterpret_cast<float4*>(M);
    float4* V4 = reinterpret_cast<float4*>(V);
    int i = threadIdx.x;
    // two float4 per thread per iteration, loads issued before the math
    for (; i + (int)blockDim.x < len4; i += 2 * blockDim.x) {
      int j = i + blockDim.x;
      float4 p0 = P4[i], g0 = G4[i], m0 = M4[i], v0 = V4[i];
      float4 p1 = P4[j], g1 = G4[j], m1 = M4[j], v1 = V4[j];
      g0 = scaled(g0);
      g1 = scaled(g1);
      adam_elem<ADAMW>(p0.x, g0.x, m0.x, v0.x, h);
      adam_elem<ADAMW>(p0.y, g0.y, m0.y, v0.y, h);
      adam_elem<ADAMW>(p0.z, g0.z, m0.z, v0.z, h);
      adam_elem<ADAMW>(p0.w, g0.w, m0.w, v0.w, h);
      adam_elem<ADAMW>(p1.x, g1.x, m1.x, v1.x, h);
      adam_elem<ADAMW>(p1.y, g1.y, m1.y, v1.y, h);
      adam_elem<ADAMW>(p1.z, g1.z, m1.z, v1.z, h);
      adam_elem<ADAMW>(p1.w, g1.w, m1.w, v1.w, h);
      P4[i] = p0; M4[i] = m0; V4[i] = v0;
      P4[j] = p1; M4[j] = m1; V4[j] = v1;
    }
    for (; i < len4; i += blockDim.x) {
      float4 p0 = P4[i], g0 = scaled(G4[i]), m0 = M4[i], v0 = V4[i];
      adam_elem<ADAMW>(p0.x, g0.x, m0.x, v0.x, h);
      adam_elem<ADAMW>(p0.y, g0.y, m0.y, v0.y, h);
      adam_elem<ADAMW>(p0.z, g0.z, m0.z, v0.z, h);
      adam_elem<ADAMW>(p0.w, g0.w, m0.w, v0.w, h);
      P4[i] = p0; M4[i] = m0; V4[i] = v0;
    }
    for (int k = (len4 << 2) + threadIdx.x; k < len; k += blockDim.x) {
      float p = P[k], m = M[k], v = V[k];
      adam_elem<ADAMW>(p, SCALED ? __fmul_rn(G[k], s) : G[k], m, v, h);
      P[k] = p; M[k] = m; V[k] = v;
    }
  }
}

struct SgdHP {
  float lr, mom, wd, omd, scale;
  int has_m, nesterov;
};

// sgd_step.wgsl:21-41; `scale` (1 for the reference op) multiplies the grad on
// read so averaged data-parallel gradients need no separate pass.
__device__ __forceinline__ void sgd_elem(float& p, float g, float& buf, const SgdHP& h) {
  if (h.scale != 1.0f) g = __fmul_rn(g, h.scale);
  if (h.wd != 0.0f) g = __fadd_rn(g, __fmul_rn(h.wd, p));
  float upd = g;
  if (h.has_m) {
    buf = __fadd_rn(__fmul_rn(buf, h.mom), __fmul_rn(g, h.omd));
    upd = h.nesterov ? __fadd_rn(g, __fmul_rn(h.mom, buf)) : buf;
  }
  p = __fsub_rn(p, __fmul_rn(h.lr, upd));
}

// x - (x with its 13 low mantissa bits cleared) per lane: the 3xTF32 low part
__device__ __forceinline__ float4 tf32_lo4(float4 v) {
  return make_float4(v.x - __uint_as_float(__float_as_uint(v.x) & 0xFFFFE000u),
                     v.y - __uint_as_float(__float_as_uint(v.y) & 0xFFFFE000u),
                     v.z - __uint_as_float(__float_as_uint(v.z) & 0xFFFFE000u),
                     v.w - __uint_as_float(__float_as_uint(v.w) & 0xFFFFE000u));
}

__global__ void __launch_bounds__(256) k_sgd_multi(const OptRow* __restrict__ rows, const OptChunk* __restrict__ chunks,
                                                   int nchunks, SgdHP h) {
  ::tp::pdl_enter();
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    OptChunk ch = chunks[c];
    OptRow r = rows[ch.row];
    float* __restrict__ P = r.p + ch.start;
    const float* __restrict__ G = r.g + ch.start;
    float* __restrict__ B = r.s0 + ch.start;
    int len = ch.len, len4 = len >> 2;
    float4* P4 = reinterpret_cast<float4*>(P);
    const float4* G4 = reinterpret_cast<const float4*>(G);
    float4* B4 = reinterpret_cast<float4*>(B);
    // the updated parameter's tf32 low parts, for rows that keep them
    float* __restrict__ LO = r.lo ? r.lo + ch.start : nullptr;
    float4* LO4 = reinterpret_cast<float4*>(LO);
    int i = threadIdx.x;
    for (; i + (int)blockDim.x < len4; i += 2 * blockDim.x) {
      int j = i + blockDim.x;
      float4 p0 = P4[i], g0 = G4[i], p1 = P4[j], g1 = G4[j];
      float4 b0 = h.has_m ? B4[i] : make_float4(0, 0, 0, 0);
      float4 b1 = h.has_m ? B4[j] : make_float4(0, 0, 0, 0);
      sgd_elem(p0.x, g0.x, b0.x, h); sgd_elem(p0.y, g0.y, b0.y, h);
      sgd_elem(p0.z, g0.z, b0.z, h); sgd_elem(p0.w, g0.w, b0.w, h);
      sgd_elem(p1.x, g1.x, b1.x, h); sgd_elem(p1.y, g1.y, b1.y, h);
      sgd_elem(p1.z, g1.z, b1.z, h); sgd_elem(p1.w, g1.w, b1.w, h);
      P4[i] = p0; P4[j] = p1;
      if (h.has_m) { B4[i] = b0; B4[j] = b1; }
      if (LO4) { LO4[i] = tf32_lo4(p0); LO4[j] = tf32_lo4(p1); }
    }
    for (; i < len4; i += blockDim.x) {
      float4 p0 = P4[i], g0 = G4[i];
      float4 b0 = h.has_m ? B4[i] : make_float4(0, 0, 0, 0);
      sgd_elem(p0.x, g0.x, b0.x, h); sgd_elem(p0.y, g0.y, b0.y, h);
      sgd_elem(p0.z, g0.z, b0.z, h); sgd_elem(p0.w, g0.w, b0.w, h);
      P4[i] = p0;
      if (h.has_m) B4[i] = b0;
      if (LO4) LO4[i] = tf32_lo4(p0);
    }
    for (int k = (len4 << 2) + threadIdx.x; k < len; k += blockDim.x) {
      float p = P[k], b = h.has_m ? B[k] : 0.0f;
      sgd_elem(p, G[k], b, h);
      P[k] = p;
      if (h.has_m) B[k] = b;
      if (LO) LO[k] = p - __uint_as_float(__float_as_uint(p) & 0xFFFFE000u);
    }
  }
}

// ---- the other fused steps (rmsprop_step.wgsl, extended_step.wgsl) ---------------------
// Same multi-tensor walk; the per-element arithmetic is each entry point's,
// operation by operation, with round-to-nearest intrinsics (no contraction), so
// the results are bit-identical to the oracle's restatement.
enum ExtKind { EXT_RMSPROP = 0, EXT_ADAGRAD = 1, EXT_ADAMAX = 2, EXT_NADAM = 3, EXT_RADAM = 4 };

struct ExtHP {
  float lr, b1, b2, eps, wd;  // RMSprop: b1 = alpha; Adagrad uses lr, eps, wd
  float step_size;            // Adamax, NAdam, RAdam
  float x0, x1;               // RMSprop: momentum; Adamax: bias_correction1; NAdam: mu;
                              // RAdam: beta1^t, beta2^t
  float t;                    // RAdam: the step count as f32 (at least 1)
  int use_momentum;           // RMSprop
};

template <int KIND>
__device__ __forceinline__ void ext_elem(float& p, float g, float& s0, float& s1, const ExtHP& h) {
  if (h.wd != 0.0f) g = __fadd_rn(g, __fmul_rn(h.wd, p));
  if (KIND == EXT_RMSPROP) {  // rmsprop_step.wgsl:22-41
    const float sq = __fadd_rn(__fmul_rn(s0, h.b1), __fmul_rn(__fmul_rn(__fsub_rn(1.0f, h.b1), g), g));
    s0 = sq;
    const float denom = __fadd_rn(__fsqrt_rn(sq), h.eps);
    float upd = __fdiv_rn(g, denom);
    if (h.use_momentum) {
      s1 = __fadd_rn(__fmul_rn(s1, h.x0), upd);
      upd = s1;
    }
    p = __fsub_rn(p, __fmul_rn(h.lr, upd));
  } else if (KIND == EXT_ADAGRAD) {  // extended_step.wgsl adagrad_step
    const float s = __fadd_rn(s0, __fmul_rn(g, g));
    s0 = s;
    const float sd = __fadd_rn(__fsqrt_rn(s), h.eps);
    p = __fsub_rn(p, __fdiv_rn(__fmul_rn(h.lr, g), sd));
  } else if (KIND == EXT_ADAMAX) {  // extended_step.wgsl adamax_step
    const float m = __fadd_rn(__fmul_rn(s0, h.b1), __fmul_rn(__fsub_rn(1.0f, h.b1), g));
    const float u = fmaxf(__fmul_rn(s1, h.b2), fabsf(g));
    s0 = m;
    s1 = u;
    const float denom = __fadd_rn(u, h.eps);
    p = __fsub_rn(p, __fmul_rn(__fmul_rn(__fdiv_rn(m, denom), h.step_size), h.x0));
  } else {
    const float m = __fadd_rn(__fmul_rn(s0, h.b1), __fmul_rn(__fsub_rn(1.0f, h.b1), g));
    const float v = __fadd_rn(__fmul_rn(s1, h.b2), __fmul_rn(__fmul_rn(__fsub_rn(1.0f, h.b2), g), g));
    s0 = m;
    s1 = v;
    if (KIND == EXT_NADAM) {  // extended_step.wgsl nadam_step
      const float m_hat = __fadd_rn(__fmul_rn(h.x0, m), __fmul_rn(__fsub_rn(1.0f, h.x0), g));
      const float denom = __fadd_rn(__fsqrt_rn(v), h.eps);
      p = __fsub_rn(p, __fmul_rn(__fdiv_rn(m_hat, denom), h.step_size));
    } else {  // extended_step.wgsl radam_step
      const float m_hat = __fdiv_rn(m, __fsub_rn(1.0f, h.x0));
      const float rho_inf = __fsub_rn(__fdiv_rn(2.0f, __fsub_rn(1.0f, h.b2)), 1.0f);
      const float omb2t = __fsub_rn(1.0f, h.x1);
      const float rho_t =
          __fsub_rn(rho_inf, __fdiv_rn(__fmul_rn(__fmul_rn(2.0f, h.t), h.x1), fmaxf(omb2t, 1e-10f)));
      float upd;
      if (rho_t > 5.0f) {
        const float num = __fmul_rn(__fmul_rn(__fsub_rn(rho_t, 4.0f), __fsub_rn(rho_t, 2.0f)), rho_inf);
        const float den = __fmul_rn(__fmul_rn(__fsub_rn(rho_inf, 4.0f), __fsub_rn(rho_inf, 2.0f)), rho_t);
        const float rect = __fsqrt_rn(__fdiv_rn(num, den));
        upd = __fmul_rn(__fmul_rn(h.step_size, m_hat), rect);
      } else {
        upd = __fmul_rn(h.step_size, m_hat);
      }
      p = __fsub_rn(p, upd);
    }
  }
}

template <int KIND>
__global__ void __launch_bounds__(256) k_ext_multi(const OptRow* __restrict__ rows, const OptChunk* __restrict__ chunks,
                                                   int nchunks, ExtHP h) {
  ::tp::pdl_enter();
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    OptChunk ch = chunks[c];
    OptRow r = rows[ch.row];
    float* __restrict__ P = r.p + ch.start;
    const float* __restrict__ G = r.g + ch.start;
    float* __restrict__ S0 = r.s0 + ch.start;
    float* __restrict__ S1 = r.s1 + ch.start;
    // Adagrad keeps one state tensor, RMSprop without momentum never touches the second
    const bool two = KIND != EXT_ADAGRAD && (KIND != EXT_RMSPROP || h.use_momentum);
    const int len = ch.len, len4 = len >> 2;
    float4* P4 = reinterpret_cast<float4*>(P);
    const float4* G4 = reinterpret_cast<const float4*>(G);
    float4* A4 = reinterpret_cast<float4*>(S0);
    float4* B4 = reinterpret_cast<float4*>(S1);
    int i = threadIdx.x;
    // two float4 per thread per iteration, all loads issued before the math
    for (; i + (int)blockDim.x < len4; i += 2 * blockDim.x) {
      const int j = i + blockDim.x;
      float4 p0 = P4[i], g0 = G4[i], a0 = A4[i], p1 = P4[j], g1 = G4[j], a1 = A4[j];
      float4 b0 = two ? B4[i] : make_float4(0, 0, 0, 0);
      float4 b1 = two ? B4[j] : make_float4(0, 0, 0, 0);
      ext_elem<KIND>(p0.x, g0.x, a0.x, b0.x, h);
      ext_elem<KIND>(p0.y, g0.y, a0.y, b0.y, h);
      ext_elem<KIND>(p0.z, g0.z, a0.z, b0.z, h);
      ext_elem<KIND>(p0.w, g0.w, a0.w, b0.w, h);
      ext_elem<KIND>(p1.x, g1.x, a1.x, b1.x, h);
      ext_elem<KIND>(p1.y, g1.y, a1.y, b1.y, h);
      ext_elem<KIND>(p1.z, g1.z, a1.z, b1.z, h);
      ext_elem<KIND>(p1.w, g1.w, a1.w, b1.w, h);
      P4[i] = p0;
      A4[i] = a0;
      P4[j] = p1;
      A4[j] = a1;
      if (two) {
        B4[i] = b0;
        B4[j] = b1;
      }
    }
    for (; i < len4; i += blockDim.x) {
      float4 p = P4[i], g = G4[i], a = A4[i];
      float4 b = two ? B4[i] : make_float4(0, 0, 0, 0);
      ext_elem<KIND>(p.x, g.x, a.x, b.x, h);
      ext_elem<KIND>(p.y, g.y, a.y, b.y, h);
      ext_elem<KIND>(p.z, g.z, a.z, b.z, h);
      ext_elem<KIND>(p.w, g.w, a.w, b.w, h);
      P4[i] = p;
      A4[i] = a;
      if (two) B4[i] = b;
    }
    for (int k = (len4 << 2) + threadIdx.x; k < len; k += blockDim.x) {
      float p = P[k], a = S0[k], b = two ? S1[k] : 0.0f;
      ext_elem<KIND>(p, G[k], a, b, h);
      P[k] = p;
      S0[k] = a;
      if (two) S1[k] = b;
    }
  }
}

// ---- the global gradient norm, and clipping ------------------------------------------
// N = (sum |g|^p)^(1/p) over every gradient of the group, p in {1, 2, inf};
// coef = min(1, max_norm / (N + 1e-6)), NaN if N is NaN (or both are infinite).
// Every CTA walks its chunks (a fixed assignment) and leaves one f64 partial;
// the next launch's CTAs each combine all partials in the same order, so equal
// inputs give equal bits and no CTA waits for another.  Squares of f32 values
// are exact in f64 and cannot overflow there.  The norm walks the chunks from
// the last to the first, the pass after it (scaling, or the step) from the first:
// what the norm read last is what that pass finds in L2.
constexpr int NORM_MAX_CTAS = 1184;

template <int P>  // 0: inf
__device__ __forceinline__ double norm_fold(double a, double b) {
  if (P != 0) return a + b;
  return (isnan(a) || a > b) ? a : b;
}
template <int P>
__device__ __forceinline__ double norm_term(float g) {
  const double d = fabs((double)g);
  return P == 2 ? d * d : d;
}

template <int P>
__device__ double norm_block(double v, double* sh) {
  for (int o = 16; o > 0; o >>= 1) v = norm_fold<P>(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v = norm_fold<P>(v, sh[w]);
  return v;
}

template <int P>
__global__ void __launch_bounds__(256) k_grad_norm(const OptRow* __restrict__ rows, const OptChunk* __restrict__ chunks,
                                                   int nchunks, int part_log, double* __restrict__ partials) {
  ::tp::pdl_enter();
  __shared__ double sh[8];
  double acc = 0.0;
  for (int c = (nchunks << part_log) - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    OptChunk ch = chunks[c >> part_log];
    if (!opt_part(ch, c, part_log)) continue;
    const float* __restrict__ G = rows[ch.row].g + ch.start;
    const float4* __restrict__ G4 = reinterpret_cast<const float4*>(G);
    const int len = ch.len, len4 = len >> 2;
    auto four = [&](float4 g) {
      return norm_fold<P>(norm_fold<P>(norm_term<P>(g.x), norm_term<P>(g.y)),
                          norm_fold<P>(norm_term<P>(g.z), norm_term<P>(g.w)));
    };
    int i = threadIdx.x;
    for (; i + 3 * 256 < len4; i += 4 * 256) {
      const float4 a = G4[i], b = G4[i + 256], c4 = G4[i + 512], d = G4[i + 768];
      acc = norm_fold<P>(acc, norm_fold<P>(norm_fold<P>(four(a), four(b)), norm_fold<P>(four(c4), four(d))));
    }
    for (; i < len4; i += 256) acc = norm_fold<P>(acc, four(G4[i]));
    for (int k = (len4 << 2) + threadIdx.x; k < len; k += 256) acc = norm_fold<P>(acc, norm_term<P>(G[k]));
  }
  acc = norm_block<P>(acc, sh);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// The norm and the coefficient from the partials; SCALE: then every gradient
// times the coefficient, left alone when it is exactly 1.
template <int P, bool SCALE>
__global__ void __launch_bounds__(256) k_grad_clip(const OptRow* __restrict__ rows, const OptChunk* __restrict__ chunks,
                                                   int nchunks, int part_log, const double* __restrict__ partials,
                                                   int np, float max_norm, float* __restrict__ out) {
  ::tp::pdl_enter();
  __shared__ double sh[8];
  double acc = 0.0;
  for (int i = threadIdx.x; i < np; i += 256) acc = norm_fold<P>(acc, partials[i]);
  acc = norm_block<P>(acc, sh);
  const double norm = P == 2 ? sqrt(acc) : acc;
  const double q = (double)max_norm / (norm + 1e-6);
  const float coef = (float)(q > 1.0 ? 1.0 : q);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    out[0] = (float)norm;
    out[1] = coef;
  }
  if (coef == 1.0f) return;
  for (int c = blockIdx.x; SCALE && c < nchunks << part_log; c += gridDim.x) {
    OptChunk ch = chunks[c >> part_log];
    if (!opt_part(ch, c, part_log)) continue;
    float* __restrict__ G = const_cast<float*>(rows[ch.row].g) + ch.start;
    float4* __restrict__ G4 = reinterpret_cast<float4*>(G);
    const int len = ch.len, len4 = len >> 2;
    auto scaled = [&](float4 g) {
      return make_float4(__fmul_rn(g.x, coef), __fmul_rn(g.y, coef), __fmul_rn(g.z, coef), __fmul_rn(g.w, coef));
    };
    int i = threadIdx.x;
    for (; i + 3 * 256 < len4; i += 4 * 256) {
      const float4 a = G4[i], b = G4[i + 256], c4 = G4[i + 512], d = G4[i + 768];
      G4[i] = scaled(a);
      G4[i + 256] = scaled(b);
      G4[i + 512] = scaled(c4);
      G4[i + 768] = scaled(d);
    }
    for (; i < len4; i += 256) G4[i] = scaled(G4[i]);
    for (int k = (len4 << 2) + threadIdx.x; k < len; k += 256) G[k] = __fmul_rn(G[k], coef);
  }
}

// ---- groups --------------------------------------------------------------------

struct Group {
  OptRow* rows = nullptr;
  OptChunk* chunks = nullptr;
  int nrows = 0;
  int nchunks = 0;
  double* partials = nullptr;   // NORM_MAX_CTAS of the gradient norm (groups built with_norm)
  bool grads_disjoint = true;   // no two rows share gradient memory: they can be scaled in place
};

static std::unordered_map<int64_t, Group> g_groups;
static int64_t g_next_group = 1;

using Span = std::pair<uintptr_t, uintptr_t>;  // of memory

static void add_span(std::vector<Span>& spans, const float* p, int64_t n) {
  if (n > 0) spans.emplace_back((uintptr_t)p, (uintptr_t)(p + n));
}

static bool disjoint(std::vector<Span> spans) {
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return false;
  return true;
}

// with_norm: with the partials and the overlap check of the gradient norm
static Group build_group(const std::vector<OptRow>& rows, bool with_norm = false) {
  // a replayed copy would read `rows` and `chunks` after they are gone
  cudaStreamCaptureStatus capture;
  TP_CUDA(cudaStreamIsCapturing(stream(), &capture));
  TP_REQUIRE(capture == cudaStreamCaptureStatusNone,
             "a list of tensors cannot be uploaded in a graph capture: create a tensor group before it");
  std::vector<OptChunk> chunks;
  for (size_t r = 0; r < rows.size(); ++r) {
    const OptRow& x = rows[r];
    TP_REQUIRE((((uintptr_t)x.p | (uintptr_t)x.g | (uintptr_t)x.s0 | (uintptr_t)x.s1 | (uintptr_t)x.lo) & 15) == 0,
               "optimizer tensors must be 16-byte aligned");
    for (int64_t s = 0; s < x.n; s += OPT_CHUNK) {
      OptChunk c;
      c.row = (int32_t)r;
      c.start = s;
      c.len = (int32_t)(x.n - s < OPT_CHUNK ? x.n - s : OPT_CHUNK);
      chunks.push_back(c);
    }
  }
  Group g;
  g.nrows = (int)rows.size();
  g.nchunks = (int)chunks.size();
  size_t rb = rows.size() * sizeof(OptRow), cb = chunks.size() * sizeof(OptChunk);
  rb = (rb + 15) & ~(size_t)15;
  char* buf = (char*)dalloc(rb + ((cb + 15) & ~(size_t)15) + (with_norm ? NORM_MAX_CTAS * sizeof(double) : 16));
  g.rows = (OptRow*)buf;
  g.chunks = (OptChunk*)(buf + rb);
  g.partials = (double*)(buf + rb + ((cb + 15) & ~(size_t)15));
  rb = rows.size() * sizeof(OptRow);
  if (rb) TP_CUDA(cudaMemcpyAsync(g.rows, rows.data(), rb, cudaMemcpyHostToDevice, stream()));
  if (cb) TP_CUDA(cudaMemcpyAsync(g.chunks, chunks.data(), cb, cudaMemcpyHostToDevice, stream()));
  if (!with_norm) return g;
  std::vector<Span> spans;
  for (const OptRow& x : rows) add_span(spans, x.g, x.n);
  g.grads_disjoint = disjoint(std::move(spans));
  return g;
}

static void free_group(Group& g) {
  dfree(g.rows);
  g.rows = nullptr;
}

static unsigned opt_grid(int nchunks) {
  unsigned cap = (unsigned)sm_count() * 4;
  return (unsigned)(nchunks < (int)cap ? (nchunks > 0 ? nchunks : 1) : cap);
}

// Parts of a chunk for a grid of 8 CTAs per SM: at most 32, 2048 values each.
static int part_log(int nchunks) {
  TP_REQUIRE(nchunks <= INT_MAX / 64, "the tensors are too many values for one launch");
  int p = 0;
  while (p < 5 && (int64_t)nchunks << p < (int64_t)sm_count() * 8) ++p;
  return p;
}

static AdamHP adam_hp(float lr, float b1, float b2, float eps, float wd, float ss, float isb) {
  AdamHP h;
  h.lr = lr; h.b1 = b1; h.b2 = b2; h.eps = eps; h.wd = wd; h.step_size = ss; h.inv_sqrt_bc2 = isb;
  h.omb1 = 1.0f - b1;  // f32 uniform arithmetic, as in the shader
  h.omb2 = 1.0f - b2;
  h.lrwd = lr * wd;
  return h;
}

void launch_adam_group(const Group& g, bool adamw, const AdamHP& h, const float* gs = nullptr) {
  if (g.nchunks == 0) return;
  const int parts = gs ? part_log(g.nchunks) : 0;
  const unsigned grid = opt_grid(g.nchunks << parts);
  if (adamw && gs) TP_LAUNCH((k_adam_multi<true, true>), grid, 256, 0, g.rows, g.chunks, g.nchunks, h, gs, parts);
  else if (adamw) TP_LAUNCH((k_adam_multi<true, false>), grid, 256, 0, g.rows, g.chunks, g.nchunks, h, gs, parts);
  else if (gs) TP_LAUNCH((k_adam_multi<false, true>), grid, 256, 0, g.rows, g.chunks, g.nchunks, h, gs, parts);
  else TP_LAUNCH((k_adam_multi<false, false>), grid, 256, 0, g.rows, g.chunks, g.nchunks, h, gs, parts);
}

void launch_sgd_group(const Group& g, const SgdHP& h) {
  if (g.nchunks == 0) return;
  TP_LAUNCH(k_sgd_multi, opt_grid(g.nchunks), 256, 0, g.rows, g.chunks, g.nchunks, h);
}

static unsigned opt_grid(int nchunks);

template <int KIND>
static void launch_ext(const Group& g, const ExtHP& h) {
  if (g.nchunks == 0) return;
  TP_LAUNCH(k_ext_multi<KIND>, opt_grid(g.nchunks), 256, 0, g.rows, g.chunks, g.nchunks, h);
}

static void launch_ext_kind(int kind, const Group& g, const ExtHP& h) {
  switch (kind) {
    case EXT_RMSPROP: launch_ext<EXT_RMSPROP>(g, h); break;
    case EXT_ADAGRAD: launch_ext<EXT_ADAGRAD>(g, h); break;
    case EXT_ADAMAX: launch_ext<EXT_ADAMAX>(g, h); break;
    case EXT_NADAM: launch_ext<EXT_NADAM>(g, h); break;
    default: launch_ext<EXT_RADAM>(g, h); break;
  }
}

// Codes of the norm: 2, 1 or inf.
static int norm_code(float norm_type, float max_norm, const char* what) {
  TP_REQUIRE(norm_type == 1.0f || norm_type == 2.0f || (std::isinf(norm_type) && norm_type > 0),
             "%s: norm_type must be 1, 2 or inf, got %g", what, (double)norm_type);
  TP_REQUIRE(max_norm >= 0.0f, "%s: max_norm must not be negative or NaN, got %g", what, (double)max_norm);
  return std::isinf(norm_type) ? 0 : (int)norm_type;
}

template <int P>
static void launch_norm(const Group& g, float max_norm, bool scale, float* out) {
  const int split = part_log(g.nchunks), items = g.nchunks << split;
  const int full = sm_count() * (split ? 8 : 4), most = full < NORM_MAX_CTAS ? full : NORM_MAX_CTAS;
  const unsigned grid = (unsigned)(items < 1 ? 1 : (items < most ? items : most));
  TP_LAUNCH(k_grad_norm<P>, grid, 256, 0, g.rows, g.chunks, g.nchunks, split, g.partials);
  if (scale) TP_LAUNCH((k_grad_clip<P, true>), grid, 256, 0, g.rows, g.chunks, g.nchunks, split, g.partials, (int)grid,
                       max_norm, out);
  else TP_LAUNCH((k_grad_clip<P, false>), 1, 256, 0, g.rows, g.chunks, g.nchunks, split, g.partials, (int)grid,
                 max_norm, out);
}

// out[0] = the norm, out[1] = the coefficient; scale: the gradients too
static void launch_grad_norm(const Group& g, int p, float max_norm, bool scale, float* out, const char* what) {
  TP_REQUIRE(!scale || g.grads_disjoint, "%s: a gradient is listed twice (or two overlap); it would be scaled twice",
             what);
  if (p == 0) launch_norm<0>(g, max_norm, scale, out);
  else if (p == 1) launch_norm<1>(g, max_norm, scale, out);
  else launch_norm<2>(g, max_norm, scale, out);
}

// Frees a call's own group, also when the call throws.
struct TempGroup {
  Group g;
  explicit TempGroup(const std::vector<OptRow>& rows) : g(build_group(rows, true)) {}
  ~TempGroup() { cudaFreeAsync(g.rows, stream()); }
};

static std::vector<OptRow> rows_from_ids(const int64_t* p, const int64_t* gr, const int64_t* s0, const int64_t* s1,
                                         int n, const char* what) {
  std::vector<OptRow> rows((size_t)n);
  for (int i = 0; i < n; ++i) {
    Tensor& tp_ = get(p[i]);
    Tensor& tg = get(gr[i]);
    Tensor& t0 = get(s0[i]);
    Tensor* t1 = s1 ? &get(s1[i]) : nullptr;
    if (tg.numel != tp_.numel || t0.numel != tp_.numel || (t1 && t1->numel != tp_.numel))
      fail(TP_ERR_ARG, "%s: tensor lengths must match", what);
    rows[i] = OptRow{tp_.f(), tg.f(), t0.f(), t1 ? t1->f() : t0.f(), nullptr, tp_.numel};
  }
  return rows;
}

}  // namespace tp

using namespace tp;

extern "C" {

TP_API int tp_adamw_step_multi(const int64_t* p, const int64_t* g, const int64_t* m, const int64_t* v, int n,
                               float lr, float b1, float b2, float eps, float wd, float ss, float isb) {
  return guard([&] {
    Group grp = build_group(rows_from_ids(p, g, m, v, n, "adamWStep"));
    launch_adam_group(grp, true, adam_hp(lr, b1, b2, eps, wd, ss, isb));
    free_group(grp);
  });
}

TP_API int tp_adam_step_multi(const int64_t* p, const int64_t* g, const int64_t* m, const int64_t* v, int n,
                              float lr, float b1, float b2, float eps, float wd, float ss, float isb) {
  return guard([&] {
    Group grp = build_group(rows_from_ids(p, g, m, v, n, "adamStep"));
    launch_adam_group(grp, false, adam_hp(lr, b1, b2, eps, wd, ss, isb));
    free_group(grp);
  });
}

TP_API int tp_adamw_step(int64_t p, int64_t g, int64_t m, int64_t v, float lr, float b1, float b2, float eps,
                         float wd, float ss, float isb) {
  return tp_adamw_step_multi(&p, &g, &m, &v, 1, lr, b1, b2, eps, wd, ss, isb);
}

TP_API int tp_adam_step(int64_t p, int64_t g, int64_t m, int64_t v, float lr, float b1, float b2, float eps, float wd,
                        float ss, float isb) {
  return tp_adam_step_multi(&p, &g, &m, &v, 1, lr, b1, b2, eps, wd, ss, isb);
}

TP_API int tp_sgd_step_multi(const int64_t* p, const int64_t* g, const int64_t* b, int n, float lr, float mom,
                             float wd, float damp, int nesterov) {
  return guard([&] {
    Group grp = build_group(rows_from_ids(p, g, b, nullptr, n, "sgdStep"));
    SgdHP h{lr, mom, wd, 1.0f - damp, 1.0f, mom != 0.0f ? 1 : 0, nesterov ? 1 : 0};
    launch_sgd_group(grp, h);
    free_group(grp);
  });
}

TP_API int tp_sgd_step(int64_t p, int64_t g, int64_t b, float lr, float mom, float wd, float damp, int nesterov) {
  return tp_sgd_step_multi(&p, &g, &b, 1, lr, mom, wd, damp, nesterov);
}

TP_API int tpk_group_create_lo(int n, float* const* params, float* const* grads, float* const* state0,
                               float* const* state1, float* const* lo, const int64_t* numels, int64_t* out_group) {
  return guard([&] {
    TP_REQUIRE(n >= 0, "negative group size");
    std::vector<OptRow> rows((size_t)n);
    for (int i = 0; i < n; ++i)
      rows[i] = OptRow{params[i], grads[i], state0[i], state1 ? state1[i] : state0[i], lo ? lo[i] : nullptr,
                       numels[i]};
    Group g = build_group(rows, true);
    int64_t id = g_next_group++;
    g_groups[id] = g;
    *out_group = id;
  });
}

TP_API int tpk_group_create(int n, float* const* params, float* const* grads, float* const* state0,
                            float* const* state1, const int64_t* numels, int64_t* out_group) {
  return tpk_group_create_lo(n, params, grads, state0, state1, nullptr, numels, out_group);
}

TP_API int tpk_group_destroy(int64_t group) {
  return guard([&] {
    auto it = g_groups.find(group);
    if (it == g_groups.end()) return;
    free_group(it->second);
    g_groups.erase(it);
  });
}

TP_API int tpk_adam_group(int64_t group, int kind, float lr, float b1, float b2, float eps, float wd, float ss,
                          float isb) {
  return guard([&] {
    auto it = g_groups.find(group);
    TP_REQUIRE(it != g_groups.end(), "unknown tensor group %lld", (long long)group);
    launch_adam_group(it->second, kind == 0, adam_hp(lr, b1, b2, eps, wd, ss, isb));
  });
}

TP_API int tpk_sgd_group(int64_t group, float lr, float mom, float wd, float damp, int nesterov, float grad_scale) {
  return guard([&] {
    auto it = g_groups.find(group);
    TP_REQUIRE(it != g_groups.end(), "unknown tensor group %lld", (long long)group);
    SgdHP h{lr, mom, wd, 1.0f - damp, grad_scale, mom != 0.0f ? 1 : 0, nesterov ? 1 : 0};
    launch_sgd_group(it->second, h);
  });
}

TP_API int tpk_group_grad_norm(int64_t group, float norm_type, float max_norm, float* norm_coef) {
  return guard([&] {
    const char* what = "group_grad_norm";
    const int p = norm_code(norm_type, max_norm, what);
    TP_REQUIRE(norm_coef, "%s: norm_coef is NULL", what);
    check_aligned({norm_coef}, what);
    auto it = g_groups.find(group);
    TP_REQUIRE(it != g_groups.end(), "unknown tensor group %lld", (long long)group);
    launch_grad_norm(it->second, p, max_norm, false, norm_coef, what);
  });
}

TP_API int tpk_group_clip_grad_norm(int64_t group, float norm_type, float max_norm, float* norm_coef) {
  return guard([&] {
    const char* what = "group_clip_grad_norm";
    const int p = norm_code(norm_type, max_norm, what);
    TP_REQUIRE(norm_coef, "%s: norm_coef is NULL", what);
    check_aligned({norm_coef}, what);
    auto it = g_groups.find(group);
    TP_REQUIRE(it != g_groups.end(), "unknown tensor group %lld", (long long)group);
    launch_grad_norm(it->second, p, max_norm, true, norm_coef, what);
  });
}

TP_API int tpk_adam_group_scaled(int64_t group, int kind, float lr, float b1, float b2, float eps, float wd, float ss,
                                 float isb, const float* grad_scale) {
  return guard([&] {
    TP_REQUIRE(kind == 0 || kind == 1, "adam_group_scaled: kind must be 0 (AdamW) or 1 (Adam), got %d", kind);
    TP_REQUIRE(grad_scale, "adam_group_scaled: grad_scale is NULL");
    check_aligned({grad_scale}, "adam_group_scaled");
    auto it = g_groups.find(group);
    TP_REQUIRE(it != g_groups.end(), "unknown tensor group %lld", (long long)group);
    launch_adam_group(it->second, kind == 0, adam_hp(lr, b1, b2, eps, wd, ss, isb), grad_scale);
  });
}

TP_API int tp_clip_grad_norm_multi(const int64_t* grads, int n, float norm_type, float max_norm, tp_handle* norm) {
  return guard([&] {
    const char* what = "clipGradNorm";
    TP_REQUIRE(n >= 0, "%s: negative tensor count", what);
    const int p = norm_code(norm_type, max_norm, what);
    std::vector<OptRow> rows((size_t)n);
    for (int i = 0; i < n; ++i) {
      const Tensor& g = get(grads[i]);
      TP_REQUIRE(g.phys == PHYS_F32, "%s: index tensors are not supported", what);
      rows[i] = OptRow{g.f(), g.f(), g.f(), g.f(), nullptr, g.numel};
    }
    TempGroup t(rows);
    Outputs o;
    const int64_t two[1] = {2};
    Tensor& out = o.add(make(two, 1, TP_FLOAT32));
    launch_grad_norm(t.g, p, max_norm, true, out.f(), what);
    o.emit_all({norm});
  });
}

TP_API int tp_adam_clip_step_multi(int kind, const int64_t* p, const int64_t* g, const int64_t* m, const int64_t* v,
                                   int n, float lr, float b1, float b2, float eps, float wd, float ss, float isb,
                                   float max_norm, tp_handle* norm) {
  return guard([&] {
    const char* what = "adamClipStep";
    TP_REQUIRE(n >= 0, "%s: negative tensor count", what);
    TP_REQUIRE(kind == 0 || kind == 1, "%s: kind must be 0 (AdamW) or 1 (Adam), got %d", what, kind);
    const int code = norm_code(2.0f, max_norm, what);
    const std::vector<OptRow> rows = rows_from_ids(p, g, m, v, n, what);
    for (int i = 0; i < n; ++i)
      TP_REQUIRE(get(p[i]).phys == PHYS_F32 && get(g[i]).phys == PHYS_F32 && get(m[i]).phys == PHYS_F32 &&
                     get(v[i]).phys == PHYS_F32,
                 "%s: index tensors are not supported", what);
    std::vector<Span> spans;
    for (const OptRow& x : rows)
      for (const float* q : {(const float*)x.p, x.g, (const float*)x.s0, (const float*)x.s1}) add_span(spans, q, x.n);
    TP_REQUIRE(disjoint(std::move(spans)), "%s: a tensor is listed twice", what);
    TempGroup t(rows);
    Outputs o;
    const int64_t two[1] = {2};
    Tensor& out = o.add(make(two, 1, TP_FLOAT32));
    launch_grad_norm(t.g, code, max_norm, false, out.f(), what);
    launch_adam_group(t.g, kind == 0, adam_hp(lr, b1, b2, eps, wd, ss, isb), out.f() + 1);
    o.emit_all({norm});
  });
}

static int ext_multi(int kind, const int64_t* p, const int64_t* g, const int64_t* s0, const int64_t* s1, int n,
                     const ExtHP& h, const char* what) {
  return guard([&] {
    TP_REQUIRE(n >= 0, "%s: negative tensor count", what);
    Group grp = build_group(rows_from_ids(p, g, s0, s1, n, what));
    launch_ext_kind(kind, grp, h);
    free_group(grp);
  });
}

static ExtHP ext_hp(float lr, float b1, float b2, float eps, float wd, float ss, float x0, float x1, float t,
                    int use_m) {
  ExtHP h;
  h.lr = lr; h.b1 = b1; h.b2 = b2; h.eps = eps; h.wd = wd; h.step_size = ss; h.x0 = x0; h.x1 = x1;
  h.t = t; h.use_momentum = use_m;
  return h;
}

TP_API int tp_rmsprop_step_multi(const int64_t* p, const int64_t* g, const int64_t* sq, const int64_t* mb, int n,
                                 float lr, float alpha, float eps, float wd, float momentum) {
  return ext_multi(EXT_RMSPROP, p, g, sq, mb, n,
                   ext_hp(lr, alpha, 0.0f, eps, wd, 0.0f, momentum, 0.0f, 0.0f, momentum != 0.0f ? 1 : 0),
                   "rmspropStep");
}

TP_API int tp_rmsprop_step(int64_t p, int64_t g, int64_t sq, int64_t mb, float lr, float alpha, float eps, float wd,
                           float momentum) {
  return tp_rmsprop_step_multi(&p, &g, &sq, &mb, 1, lr, alpha, eps, wd, momentum);
}

TP_API int tp_adagrad_step_multi(const int64_t* p, const int64_t* g, const int64_t* sum, int n, float lr, float eps,
                                 float wd) {
  return ext_multi(EXT_ADAGRAD, p, g, sum, nullptr, n, ext_hp(lr, 0.0f, 0.0f, eps, wd, 0.0f, 0.0f, 0.0f, 0.0f, 0),
                   "adagradStep");
}

TP_API int tp_adagrad_step(int64_t p, int64_t g, int64_t sum, float lr, float eps, float wd) {
  return tp_adagrad_step_multi(&p, &g, &sum, 1, lr, eps, wd);
}

TP_API int tp_adamax_step_multi(const int64_t* p, const int64_t* g, const int64_t* m, const int64_t* u, int n,
                                float lr, float b1, float b2, float eps, float wd, float step_size, float bc1) {
  return ext_multi(EXT_ADAMAX, p, g, m, u, n, ext_hp(lr, b1, b2, eps, wd, step_size, bc1, 0.0f, 0.0f, 0),
                   "adamaxStep");
}

TP_API int tp_adamax_step(int64_t p, int64_t g, int64_t m, int64_t u, float lr, float b1, float b2, float eps,
                          float wd, float step_size, float bc1) {
  return tp_adamax_step_multi(&p, &g, &m, &u, 1, lr, b1, b2, eps, wd, step_size, bc1);
}

TP_API int tp_nadam_step_multi(const int64_t* p, const int64_t* g, const int64_t* m, const int64_t* v, int n,
                               float lr, float b1, float b2, float eps, float wd, float step_size, float mu) {
  return ext_multi(EXT_NADAM, p, g, m, v, n, ext_hp(lr, b1, b2, eps, wd, step_size, mu, 0.0f, 0.0f, 0),
                   "nadamStep");
}

TP_API int tp_nadam_step(int64_t p, int64_t g, int64_t m, int64_t v, float lr, float b1, float b2, float eps,
                         float wd, float step_size, float mu) {
  return tp_nadam_step_multi(&p, &g, &m, &v, 1, lr, b1, b2, eps, wd, step_size, mu);
}

TP_API int tp_radam_step_multi(const int64_t* p, const int64_t* g, const int64_t* m, const int64_t* v, int n,
                               float lr, float b1, float b2, float eps, float wd, float step_size, float b1pow,
                               float b2pow, int64_t step) {
  const float t = (float)(step > 1 ? (uint32_t)step : 1u);  // max(f32(u32 step), 1.0)
  return ext_multi(EXT_RADAM, p, g, m, v, n, ext_hp(lr, b1, b2, eps, wd, step_size, b1pow, b2pow, t, 0),
                   "radamStep");
}

TP_API int tp_radam_step(int64_t p, int64_t g, int64_t m, int64_t v, float lr, float b1, float b2, float eps,
                         float wd, float step_size, float b1pow, float b2pow, int64_t step) {
  return tp_radam_step_multi(&p, &g, &m, &v, 1, lr, b1, b2, eps, wd, step_size, b1pow, b2pow, step);
}

}  // extern "C"
