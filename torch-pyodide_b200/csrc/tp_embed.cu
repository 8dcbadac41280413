// Rows of a table by token id, scaled, and the table's gradient.
//
//   out_i = scale * table[id_i]         dtable_v (+)= scale * sum over { i : id_i = v } of dout_i
//
// Both move bytes and add little: what bounds them is HBM.  The gradient's sum
// runs in an order fixed by the positions alone (no float atomics), so equal
// inputs give equal bits.
#include <cuda_runtime.h>

#include <climits>

#include "tp_core.h"
#include "tp_fastdiv.cuh"
#include "tp_launch.h"
#include "tp_token.cuh"

namespace tp {

// A column of a row: 4 values where rows start on 16-byte boundaries, else 1.
template <int VEC>
struct Col;
template <>
struct Col<4> {
  float4 v;
  __device__ static Col zero() { return {make_float4(0.0f, 0.0f, 0.0f, 0.0f)}; }
  __device__ __forceinline__ void add(const Col& o) { v.x += o.v.x, v.y += o.v.y, v.z += o.v.z, v.w += o.v.w; }
  __device__ __forceinline__ Col times(float s) const { return {make_float4(v.x * s, v.y * s, v.z * s, v.w * s)}; }
  __device__ static Col load(const float* p, int64_t c) { return {*(reinterpret_cast<const float4*>(p) + c)}; }
  __device__ void store(float* p, int64_t c) const { *(reinterpret_cast<float4*>(p) + c) = v; }
};
template <>
struct Col<1> {
  float v;
  __device__ static Col zero() { return {0.0f}; }
  __device__ __forceinline__ void add(const Col& o) { v += o.v; }
  __device__ __forceinline__ Col times(float s) const { return {v * s}; }
  __device__ static Col load(const float* p, int64_t c) { return {p[c]}; }
  __device__ void store(float* p, int64_t c) const { p[c] = v; }
};

// CTAs of 128 threads, `tx` across a row's columns and the rest across rows.
constexpr int EMB_NT = 128;
static int block_cols(int64_t cols) {
  int tx = 1;
  while (tx < EMB_NT && tx < cols) tx *= 2;
  return tx;
}

// ---- lookup ---------------------------------------------------------------------------
constexpr int EMB_U = 4;  // columns per thread, loaded before the first is stored

template <int VEC>
__global__ void __launch_bounds__(EMB_NT) k_embed(const float* __restrict__ table, int64_t ld,
                                                  const void* __restrict__ ids, int kind, int64_t n, int64_t V,
                                                  int64_t cols, int chunks, float scale, float* __restrict__ out,
                                                  int64_t ldo) {
  ::tp::pdl_enter();
  const int64_t group = blockIdx.x / chunks;
  const int64_t i = group * blockDim.y + threadIdx.y;
  const int64_t c0 = (int64_t)(blockIdx.x - group * chunks) * EMB_U * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t v = token_id(ids, kind, i);
  const bool in = v >= 0 && v < V;
  const float* src = table + v * ld;
  float* dst = out + i * ldo;
  Col<VEC> x[EMB_U];
#pragma unroll
  for (int u = 0; u < EMB_U; ++u) {
    const int64_t c = c0 + u * (int)blockDim.x;
    if (in && c < cols) x[u] = Col<VEC>::load(src, c);
  }
#pragma unroll
  for (int u = 0; u < EMB_U; ++u) {
    const int64_t c = c0 + u * (int)blockDim.x;
    if (c < cols) (in ? x[u].times(scale) : Col<VEC>::zero().times(NAN)).store(dst, c);
  }
}

// ---- gradient of a few tokens ---------------------------------------------------------
// One CTA per (position, 256 columns): the first position of a token sums all
// of them, in order.  Reads the ids n times over, which for few is less than
// sorting them costs.
__global__ void __launch_bounds__(256) k_embed_bwd_few(const float* __restrict__ dout, int64_t ldo,
                                                       const void* __restrict__ ids, int kind, int n, int64_t V,
                                                       int64_t D, int chunks, float scale, int64_t pad,
                                                       float* __restrict__ dtable, int64_t ld) {
  ::tp::pdl_enter();
  __shared__ uint32_t hit[8];
  const int i = blockIdx.x / chunks;
  const int64_t d = (int64_t)(blockIdx.x - i * chunks) * 256 + threadIdx.x;
  const int64_t v = token_id(ids, kind, i);
  if (v < 0 || v >= V || v == pad) return;
  bool earlier = false;
  for (int j = threadIdx.x; j < i; j += 256) earlier |= token_id(ids, kind, j) == v;
  if (__syncthreads_or(earlier)) return;
  float acc = 0.0f;
  for (int j0 = i; j0 < n; j0 += 256) {
    const int j = j0 + threadIdx.x;
    const uint32_t b = __ballot_sync(0xffffffffu, j < n && token_id(ids, kind, j) == v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) hit[threadIdx.x >> 5] = b;
    __syncthreads();
    float part = 0.0f;  // chains of at most 256 additions, then of n / 256
    for (int w = 0; w < 8; ++w)
      for (uint32_t q = hit[w]; q; q &= q - 1)
        if (d < D) part += dout[(int64_t)(j0 + 32 * w + __ffs(q) - 1) * ldo + d];
    acc += part;
  }
  if (d < D) dtable[v * ld + d] += acc * scale;
}

// ---- gradient of many tokens: positions sorted by token, then summed -----------------------
// Sorting is one launch of CTAs that share nothing.  Token v belongs to CTA
// v mod G, as its token v / G (neighbouring ids, of like frequency, go to
// different CTAs).  Each CTA reads all ids: it counts those of the CTAs before
// it, which is where its own begin, and the tokens of its own per warp; after a
// scan over (token, warp) the warps place their positions in order.  A position
// and its token are written per valid id, the start of each token's run per
// token.  (Reading all ids G times is n G 4 bytes from L2; the rows they stand for
// are n D 4 bytes from HBM.)
constexpr int SORT_NT = 1024;
constexpr int SORT_WARPS = SORT_NT / 32;
constexpr int SORT_TOKENS = 512;          // tokens of one CTA, at most
constexpr int SORT_WORDS = 32768;         // positions / 32 whose hits are kept in shared memory
constexpr int SORT_U = 16;                // ids of a thread in flight

struct EmbedSort {
  FastDiv ctas;   // G
  int per;        // tokens of one CTA, W
  int64_t n;
  int V, pad, kind;
  const void* ids;
  int32_t* start;  // [G W + 1]: where the run of key owner * W + local starts; the last: how many positions there are
  int32_t* pos;    // [n]
  int32_t* tok;    // [n]
  __device__ __forceinline__ bool valid(int v) const { return v >= 0 && v < V && v != pad; }
  __device__ __forceinline__ int key(int v) const {
    const int q = (int)ctas.div((uint32_t)v);
    return (v - q * (int)ctas.d) * per + q;
  }
  __device__ __forceinline__ int total() const { return start[(int64_t)ctas.d * per]; }
};

__global__ void __launch_bounds__(SORT_NT) k_embed_sort(const EmbedSort e) {
  ::tp::pdl_enter();
  extern __shared__ int32_t sort_sm[];
  __shared__ int32_t sh[SORT_WARPS], hits[SORT_WARPS][64];
  const int W = e.per, me = blockIdx.x, t = threadIdx.x, lane = t & 31, w = t >> 5;
  int32_t* count = sort_sm;                                  // [warps][W]
  uint32_t* words = (uint32_t*)(sort_sm + SORT_WARPS * W);   // hits of 32 positions each
  const int64_t nwords = (e.n + 31) >> 5;
  const bool kept = nwords <= SORT_WORDS;
  const int64_t per = (nwords + SORT_WARPS - 1) / SORT_WARPS;  // words of one warp: neighbours, so that order is kept
  const int64_t w0 = per * w < nwords ? per * w : nwords, w1 = w0 + per < nwords ? w0 + per : nwords;
  for (int i = t; i < SORT_WARPS * W; i += SORT_NT) count[i] = 0;
  __syncthreads();
  auto token = [&](int64_t word) {
    const int64_t p = word * 32 + lane;
    return word < w1 && p < e.n ? token_id(e.ids, e.kind, p) : -1;
  };
  int less = 0;
  for (int64_t i = w0; i < w1; i += SORT_U) {
    int v[SORT_U];
#pragma unroll
    for (int q = 0; q < SORT_U; ++q) v[q] = token(i + q);
#pragma unroll
    for (int q = 0; q < SORT_U; ++q) {
      const bool ok = e.valid(v[q]);
      const int local = (int)e.ctas.div(ok ? (uint32_t)v[q] : 0u), owner = v[q] - local * (int)e.ctas.d;
      less += ok && owner < me;
      const bool hit = ok && owner == me;
      if (hit) atomicAdd(&count[w * W + local], 1);
      const uint32_t b = __ballot_sync(0xffffffffu, hit);
      if (kept && lane == 0 && i + q < w1) words[i + q] = b;
    }
  }
  for (int o = 16; o > 0; o >>= 1) less += __shfl_xor_sync(0xffffffffu, less, o);
  if (lane == 0) sh[w] = less;
  __syncthreads();
  int base = 0;
  for (int i = 0; i < SORT_WARPS; ++i) base += sh[i];
  __syncthreads();
  // one thread per token: its warps' counts become the places of their positions
  int k[SORT_WARPS], c = 0;
  if (t < W)
#pragma unroll
    for (int i = 0; i < SORT_WARPS; ++i) k[i] = count[i * W + t];
  if (t < W)
#pragma unroll
    for (int i = 0; i < SORT_WARPS; ++i) c += k[i];
  int incl = c;  // scan over the tokens
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) sh[w] = incl;
  __syncthreads();
  int first = base + incl - c;
  for (int i = 0; i < w; ++i) first += sh[i];
  if (t < W) {
    e.start[(int64_t)me * W + t] = first;
    int at = first;
#pragma unroll
    for (int i = 0; i < SORT_WARPS; ++i) {
      count[i * W + t] = at;
      at += k[i];
    }
    if (me == (int)gridDim.x - 1 && t == W - 1) e.start[(int64_t)gridDim.x * W] = first + c;
  }
  __syncthreads();
  // Positions of hits, in order, 32 at a time: a lane each.
  int32_t* buf = hits[w];
  int have = 0;
  auto place = [&](int k) {  // the first k of buf
    __syncwarp();
    const uint32_t some = k == 32 ? 0xffffffffu : (1u << k) - 1;
    if (lane < k) {
      const int p = buf[lane], v = token_id(e.ids, e.kind, p), local = (int)e.ctas.div((uint32_t)v);
      const uint32_t peers = __match_any_sync(some, local);
      const int rank = __popc(peers & ((1u << lane) - 1)), at = count[w * W + local];
      __syncwarp(some);
      if (rank == 0) count[w * W + local] = at + __popc(peers);
      e.pos[at + rank] = p;
      e.tok[at + rank] = v;
    }
    __syncwarp();
  };
  auto take = [&](int64_t word, uint32_t b) {
    if (b >> lane & 1) buf[have + __popc(b & ((1u << lane) - 1))] = (int32_t)(word * 32 + lane);
    have += __popc(b);
    if (have >= 32) {
      place(32);
      const int32_t rest = buf[32 + lane];
      __syncwarp();
      buf[lane] = rest;
      have -= 32;
      __syncwarp();
    }
  };
  if (kept) {
    for (int64_t i = w0; i < w1; i += 32) {
      const uint32_t mine = i + lane < w1 ? words[i + lane] : 0u;
      for (uint32_t some = __ballot_sync(0xffffffffu, mine != 0u); some; some &= some - 1) {
        const int j = __ffs(some) - 1;
        take(i + j, __shfl_sync(0xffffffffu, mine, j));
      }
    }
  } else {
    for (int64_t i = w0; i < w1; ++i) {
      const int v = token(i);
      const bool ok = e.valid(v);
      take(i, __ballot_sync(0xffffffffu, ok && (int)e.ctas.mod(ok ? (uint32_t)v : 0u) == me));
    }
  }
  if (have) place(have);
}

// Tiles of SUM_T sorted positions are summed each by itself, so a frequent
// token takes no longer than many rare ones.  A run (the positions of one token)
// of at most SUM_RUN goes whole to the tile it starts in.  A longer one is cut
// at the tiles' borders: what came in from the tile before is the tile's
// partial 0, the start of what goes on its partial 1 (what does both, partial 0).
constexpr int SUM_T = 64, SUM_RUN = 128;
constexpr int SUM_ZERO = 4;  // rows without a token that a thread clears

template <int VEC, bool ACC>
__global__ void __launch_bounds__(EMB_NT) k_embed_sum(const EmbedSort e, const float* __restrict__ dout, int64_t ldo,
                                                      int64_t cols, int chunks, int64_t tiles, int64_t tile_ctas,
                                                      float scale, float* __restrict__ dtable, int64_t ld,
                                                      float* __restrict__ partial, int64_t ldp,
                                                      int2* __restrict__ cut) {
  ::tp::pdl_enter();
  const int64_t group = blockIdx.x / chunks;
  const int64_t c = (int64_t)(blockIdx.x - group * chunks) * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  if (group >= tile_ctas) {  // rows whose token is absent
    const int64_t v0 = ((group - tile_ctas) * blockDim.y + threadIdx.y) * SUM_ZERO;
#pragma unroll
    for (int r = 0; r < SUM_ZERO; ++r) {
      const int64_t v = v0 + r;
      if (v >= e.V) return;
      const int k = e.key((int)v);
      if (e.start[k] == e.start[k + 1]) Col<VEC>::zero().store(dtable + v * ld, c);
    }
    return;
  }
  const int64_t tile = group * blockDim.y + threadIdx.y;
  const int m = e.total();
  int2 starts = make_int2(-1, 0);  // the cut run that starts here: its token, its last tile
  if (tile * SUM_T >= m) {
    if (c == 0 && tile < tiles) cut[tile] = starts;
    return;
  }
  const int s0 = (int)(tile * SUM_T);
  int s1 = m - s0 < SUM_T ? m : s0 + SUM_T, from = s0;
  int cur = e.tok[s0];
  bool came_in = false, goes_on = false;
  if (s0 > 0 && e.tok[s0 - 1] == cur) {
    const int k = e.key(cur), end = e.start[k + 1];
    if (end - e.start[k] > SUM_RUN) came_in = true;
    else from = end;
  }
  if (s1 < m) {
    const int v = e.tok[s1 - 1];
    if (e.tok[s1] == v) {
      const int k = e.key(v), end = e.start[k + 1];
      if (end - e.start[k] > SUM_RUN) {
        goes_on = true;
        if (e.start[k] >= s0) starts = make_int2(v, (end - 1) / SUM_T);
      } else if (e.start[k] >= s0) {
        s1 = end;
      }
    }
  }
  if (c == 0) cut[tile] = starts;
  if (from >= s1) return;  // all of it belongs to a run of the tile before
  cur = e.tok[from];
  float* part = partial + 2 * tile * ldp;
  Col<VEC> acc = Col<VEC>::zero();
  auto flush = [&]() {
    if (came_in) {
      acc.store(part, c);
    } else {
      float* row = dtable + (int64_t)cur * ld;
      Col<VEC> r = acc.times(scale);
      if (ACC) r.add(Col<VEC>::load(row, c));
      r.store(row, c);
    }
  };
  for (int s = from; s < s1; s += 8) {
    int tok[8];
    Col<VEC> x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s + k < s1) {
        tok[k] = e.tok[s + k];
        x[k] = Col<VEC>::load(dout + (int64_t)e.pos[s + k] * ldo, c);
      }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s + k < s1) {
        if (tok[k] != cur) {
          flush();
          cur = tok[k];
          came_in = false;
          acc = Col<VEC>::zero();
        }
        acc.add(x[k]);
      }
  }
  if (!came_in && goes_on) acc.store(part + ldp, c);
  else flush();
}

// The runs that were cut: the tile one starts in adds up its partial 1 and the
// partials 0 of the tiles after it, in f64: eight threads take every eighth,
// and their sums are added in order.  A CTA looks through 32 tiles for such starts.
constexpr int JOIN_COLS = 32, JOIN_ROWS = 8;

template <bool ACC>
__global__ void __launch_bounds__(JOIN_COLS* JOIN_ROWS) k_embed_join(const int2* __restrict__ cut,
                                                                     int64_t tiles, int64_t D, int chunks,
                                                                     float scale, float* __restrict__ dtable,
                                                                     int64_t ld, const float* __restrict__ partial,
                                                                     int64_t ldp) {
  ::tp::pdl_enter();
  __shared__ double sh[JOIN_ROWS][JOIN_COLS];
  const int64_t group = blockIdx.x / chunks;
  const int64_t c = (int64_t)(blockIdx.x - group * chunks) * JOIN_COLS + threadIdx.x;
  const int64_t mine = group * 32 + threadIdx.x;  // every warp looks at the same 32 tiles
  const int2 run = mine < tiles ? cut[mine] : make_int2(-1, 0);
  for (uint32_t some = __ballot_sync(0xffffffffu, run.x >= 0); some; some &= some - 1) {
    const int which = __ffs(some) - 1;
    const int64_t tile = group * 32 + which;
    const int v = __shfl_sync(0xffffffffu, run.x, which), last = __shfl_sync(0xffffffffu, run.y, which);
    double acc = 0.0;
    if (c < D) {
      if (threadIdx.y == 0) acc = partial[(2 * tile + 1) * ldp + c];
#pragma unroll 8
      for (int64_t k = tile + 1 + threadIdx.y; k <= last; k += JOIN_ROWS) acc += partial[2 * k * ldp + c];
    }
    sh[threadIdx.y][threadIdx.x] = acc;
    __syncthreads();
    if (threadIdx.y == 0 && c < D) {
      for (int r = 1; r < JOIN_ROWS; ++r) acc += sh[r][threadIdx.x];
      float* row = dtable + (int64_t)v * ld;
      const float g = (float)(acc * scale);
      row[c] = ACC ? row[c] + g : g;
    }
    __syncthreads();
  }
}

// ---- launches -----------------------------------------------------------------------------
static bool aligned_rows(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && (ld & 3) == 0; }

static unsigned grid_of(int64_t groups, int64_t chunks, const char* what) {
  TP_REQUIRE(groups <= INT_MAX / chunks, "%s: too many tokens, rows or columns for one launch", what);
  return (unsigned)(groups * chunks);
}

void launch_embed(const float* table, int64_t ld, const void* ids, int kind, int64_t n, int64_t V, int64_t D,
                  float scale, float* out, int64_t ldo) {
  if (n == 0 || D == 0) return;
  const bool vec = D % 4 == 0 && aligned_rows(table, ld) && aligned_rows(out, ldo);
  const int64_t cols = vec ? D / 4 : D;
  const int tx = block_cols((cols + EMB_U - 1) / EMB_U), ty = EMB_NT / tx;
  const int chunks = (int)((cols + EMB_U * tx - 1) / (EMB_U * tx));
  const unsigned grid = grid_of((n + ty - 1) / ty, chunks, "token_embedding");
  if (vec) TP_LAUNCH(k_embed<4>, grid, dim3(tx, ty), 0, table, ld, ids, kind, n, V, cols, chunks, scale, out, ldo);
  else TP_LAUNCH(k_embed<1>, grid, dim3(tx, ty), 0, table, ld, ids, kind, n, V, cols, chunks, scale, out, ldo);
}

// Up to this many tokens are added to an existing gradient without sorting.
constexpr int64_t EMB_FEW = 2048;

struct EmbedPlan {
  int64_t ctas, per, start, pos, tok, cut, partial, ldp, bytes, tiles;
  EmbedPlan(int64_t n, int64_t V, int64_t D) {
    const int64_t sms = 148, waves = (V + sms * SORT_TOKENS - 1) / (sms * SORT_TOKENS);
    ctas = V < sms * waves ? V : sms * waves;
    per = (V + ctas - 1) / ctas;
    tiles = (n + SUM_T - 1) / SUM_T;
    ldp = (D + 3) / 4 * 4;
    auto up = [](int64_t b) { return (b + 15) / 16 * 16; };
    start = 0;
    pos = start + up((ctas * per + 1) * 4);
    tok = pos + up(n * 4);
    cut = tok + up(n * 4);
    partial = cut + up(tiles * 8);
    bytes = partial + 2 * tiles * ldp * 4;
  }
};

int64_t embed_bwd_ws(int64_t n, int64_t V, int64_t D) { return EmbedPlan(n, V, D).bytes; }

template <int VEC, bool ACC>
static void launch_sum(const EmbedPlan& p, const EmbedSort& e, const float* dout, int64_t ldo, int64_t D, float scale,
                       float* dtable, int64_t ld, float* partial, int2* cut) {
  const char* what = "token_embedding_backward";
  const int64_t cols = VEC == 4 ? D / 4 : D;
  const int tx = block_cols(cols), ty = EMB_NT / tx;
  const int chunks = (int)((cols + tx - 1) / tx);
  const int64_t tile_ctas = (p.tiles + ty - 1) / ty;
  const int64_t zero_ctas = ACC ? 0 : ((int64_t)e.V + ty * SUM_ZERO - 1) / (ty * SUM_ZERO);
  const unsigned grid = grid_of(tile_ctas + zero_ctas, chunks, what);
  if (grid == 0) return;
  TP_LAUNCH((k_embed_sum<VEC, ACC>), grid, dim3(tx, ty), 0, e, dout, ldo, cols, chunks, p.tiles, tile_ctas, scale,
            dtable, ld, partial, p.ldp, cut);
  if (p.tiles < 2) return;  // nothing crosses
  const int jchunks = (int)((D + JOIN_COLS - 1) / JOIN_COLS);
  TP_LAUNCH(k_embed_join<ACC>, grid_of((p.tiles + 31) / 32, jchunks, what), dim3(JOIN_COLS, JOIN_ROWS), 0,
            cut, p.tiles, D, jchunks, scale, dtable, ld, partial, p.ldp);
}

void launch_embed_bwd(const float* dout, int64_t ldo, const void* ids, int kind, int64_t n, int64_t V, int64_t D,
                      float scale, int64_t pad, bool accumulate, float* dtable, int64_t ld, void* ws) {
  if (D == 0 || (n == 0 && accumulate)) return;
  if (accumulate && n <= EMB_FEW) {
    const int chunks = (int)((D + 255) / 256);
    TP_LAUNCH(k_embed_bwd_few, grid_of(n, chunks, "token_embedding_backward"), 256, 0, dout, ldo, ids, kind, (int)n, V,
              D, chunks, scale, pad, dtable, ld);
    return;
  }
  const EmbedPlan p(n, V, D);
  char* base = (char*)ws;
  EmbedSort e;
  e.ctas = fast_div((uint32_t)p.ctas);
  e.per = (int)p.per;
  e.n = n;
  e.V = (int)V;
  e.pad = (int)pad;
  e.kind = kind;
  e.ids = ids;
  e.start = (int32_t*)(base + p.start);
  e.pos = (int32_t*)(base + p.pos);
  e.tok = (int32_t*)(base + p.tok);
  float* partial = (float*)(base + p.partial);
  int2* cut = (int2*)(base + p.cut);
  const int64_t words = (n + 31) / 32;
  const size_t smem = (size_t)(SORT_WARPS * p.per + (words <= SORT_WORDS ? words : 0)) * 4;
  static bool raised = false;
  if (!raised) {  // 64 KB of counts and 128 KB of hits at most
    TP_CUDA(cudaFuncSetAttribute(k_embed_sort, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (SORT_WARPS * SORT_TOKENS + SORT_WORDS) * 4));
    raised = true;
  }
  TP_LAUNCH(k_embed_sort, (unsigned)p.ctas, SORT_NT, smem, e);
  const bool vec = D % 4 == 0 && aligned_rows(dout, ldo) && aligned_rows(dtable, ld);
  if (vec && accumulate) launch_sum<4, true>(p, e, dout, ldo, D, scale, dtable, ld, partial, cut);
  else if (vec) launch_sum<4, false>(p, e, dout, ldo, D, scale, dtable, ld, partial, cut);
  else if (accumulate) launch_sum<1, true>(p, e, dout, ldo, D, scale, dtable, ld, partial, cut);
  else launch_sum<1, false>(p, e, dout, ldo, D, scale, dtable, ld, partial, cut);
}

static void check_embed(int64_t n, int64_t V, int64_t D, int64_t ld, int64_t ldo, const char* what) {
  TP_REQUIRE(n >= 0 && n < INT_MAX, "%s: %lld tokens is outside [0, 2^31 - 1)", what, (long long)n);
  check_vocab(V, what);
  TP_REQUIRE(D >= 0 && D <= INT_MAX, "%s: a width of %lld is outside [0, 2^31)", what, (long long)D);
  TP_REQUIRE(ld >= D && ldo >= D, "%s: a row stride (%lld, %lld) is shorter than the width %lld", what, (long long)ld,
             (long long)ldo, (long long)D);
}

}  // namespace tp

using namespace tp;

extern "C" {

TP_API int tpk_token_embedding(const float* table, int64_t ld, const void* ids, int ids_kind, int64_t n,
                               int64_t vocab, int64_t dim, float scale, float* out, int64_t ldo) {
  return guard([&] {
    const char* what = "token_embedding";
    check_embed(n, vocab, dim, ld, ldo, what);
    check_ids_kind(ids_kind, what);
    if (n == 0 || dim == 0) return;
    TP_REQUIRE(table && ids && out, "%s: table, ids and out must not be NULL", what);
    TP_REQUIRE((((uintptr_t)table | (uintptr_t)ids | (uintptr_t)out) & 3) == 0, "%s: a buffer is not 4-byte aligned",
               what);
    launch_embed(table, ld, ids, ids_kind, n, vocab, dim, scale, out, ldo);
  });
}

TP_API int tpk_token_embedding_backward_ws(int64_t n, int64_t vocab, int64_t dim, int64_t* bytes) {
  return guard([&] {
    check_embed(n, vocab, dim, dim, dim, "token_embedding_backward_ws");
    TP_REQUIRE(bytes, "token_embedding_backward_ws: bytes is NULL");
    *bytes = embed_bwd_ws(n, vocab, dim);
  });
}

TP_API int tpk_token_embedding_backward(const float* dout, int64_t ldo, const void* ids, int ids_kind, int64_t n,
                                        int64_t vocab, int64_t dim, float scale, int64_t padding_id, int accumulate,
                                        float* dtable, int64_t ld, void* ws, int64_t ws_bytes) {
  return guard([&] {
    const char* what = "token_embedding_backward";
    check_embed(n, vocab, dim, ld, ldo, what);
    check_ids_kind(ids_kind, what);
    TP_REQUIRE(padding_id >= -1 && padding_id < vocab, "%s: padding_id %lld is neither -1 nor a row of the table",
               what, (long long)padding_id);
    TP_REQUIRE(accumulate == 0 || accumulate == 1, "%s: accumulate must be 0 or 1, got %d", what, accumulate);
    if (dim == 0) return;
    TP_REQUIRE(dtable && (n == 0 || (dout && ids)), "%s: dout, ids and dtable must not be NULL", what);
    TP_REQUIRE((((uintptr_t)dout | (uintptr_t)ids | (uintptr_t)dtable) & 3) == 0,
               "%s: a buffer is not 4-byte aligned", what);
    const int64_t need = embed_bwd_ws(n, vocab, dim);
    TP_REQUIRE(ws_bytes >= need && (need == 0 || ws), "%s: a workspace of %lld bytes, %lld are needed", what,
               (long long)ws_bytes, (long long)need);
    TP_REQUIRE(((uintptr_t)ws & 15) == 0, "%s: the workspace is not 16-byte aligned", what);
    launch_embed_bwd(dout, ldo, ids, ids_kind, n, vocab, dim, scale, padding_id, accumulate != 0, dtable, ld, ws);
  });
}

TP_API int tp_token_embedding(int64_t table, int64_t ids, float scale, tp_handle* out) {
  return guard([&] {
    const char* what = "tokenEmbedding";
    const Tensor T = get(table), I = get(ids);
    TP_REQUIRE(T.ndim == 2 && T.phys == PHYS_F32, "%s: expects a float table [vocab, dim]", what);
    TP_REQUIRE(I.ndim < TP_MAX_DIMS, "%s: ids of rank %d leave no dim for the rows", what, I.ndim);
    check_embed(I.numel, T.shape[0], T.shape[1], T.shape[1], T.shape[1], what);
    std::vector<int64_t> s = shape_of(I);
    s.push_back(T.shape[1]);
    Outputs o;
    Tensor& y = o.add(make_like_shape(s, T.dtype));
    launch_embed(T.f(), T.shape[1], I.ptr, ids_kind_of(I), I.numel, T.shape[0], T.shape[1], scale, y.f(), T.shape[1]);
    o.emit_all({out});
  });
}

TP_API int tp_token_embedding_backward(int64_t grad_out, int64_t ids, int64_t vocab, float scale, int64_t padding_id,
                                       int64_t into, tp_handle* out) {
  return guard([&] {
    const char* what = "tokenEmbeddingBackward";
    const Tensor G = get(grad_out), I = get(ids);
    TP_REQUIRE(G.ndim >= 1 && G.phys == PHYS_F32, "%s: expects a float gradient [..., dim]", what);
    const int64_t n = I.numel, D = G.shape[G.ndim - 1];
    TP_REQUIRE(n * D == G.numel, "%s: %lld token ids for a gradient of %lld values in rows of %lld", what,
               (long long)n, (long long)G.numel, (long long)D);
    check_embed(n, vocab, D, D, D, what);
    TP_REQUIRE(padding_id >= -1 && padding_id < vocab, "%s: padding_id %lld is neither -1 nor a row of the table",
               what, (long long)padding_id);
    const Tensor T = into ? get(into) : Tensor();
    TP_REQUIRE(!into || (T.ndim == 2 && T.shape[0] == vocab && T.shape[1] == D && T.phys == PHYS_F32),
               "%s: the gradient to add to is not a float [%lld, %lld]", what, (long long)vocab, (long long)D);
    TP_REQUIRE(!into || (into != grad_out && into != ids), "%s: the gradient to add to is an input", what);
    Outputs o, tmp;
    const int64_t s[2] = {vocab, D}, w[1] = {(embed_bwd_ws(n, vocab, D) + 3) / 4};
    const Tensor ws = tmp.add(make(w, 1, TP_FLOAT32));
    const Tensor dt = into ? T : o.add(make(s, 2, G.dtype));
    launch_embed_bwd(G.f(), D, I.ptr, ids_kind_of(I), n, vocab, D, scale, padding_id, into != 0, dt.f(), D, ws.ptr);
    if (into) fill_handle(T, into, out);
    else o.emit_all({out});
  });
}

}  // extern "C"
