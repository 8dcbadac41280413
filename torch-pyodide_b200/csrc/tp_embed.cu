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
#include "tp_launch.h"
#include "tp_token.cuh"

namespace tp {

// A column of a row: 4 values where rows start on 16-byte boundaries, 2 where they
// do on 8-byte ones, else 1.
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
struct Col<2> {
  float2 v;
  __device__ static Col zero() { return {make_float2(0.0f, 0.0f)}; }
  __device__ __forceinline__ void add(const Col& o) { v.x += o.v.x, v.y += o.v.y; }
  __device__ __forceinline__ Col times(float s) const { return {make_float2(v.x * s, v.y * s)}; }
  __device__ static Col load(const float* p, int64_t c) { return {*(reinterpret_cast<const float2*>(p) + c)}; }
  __device__ void store(float* p, int64_t c) const { *(reinterpret_cast<float2*>(p) + c) = v; }
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
// A row to up to 128 threads of a CTA, several columns each, all loaded before the
// first is stored; the rest of its 256 threads take other rows, since SMs start
// CTAs only so fast (85921 x 535 by CTAs of one row 178 us, of 4 rows 54).  Offsets
// are 32-bit and step by the CTA's width: rows that are no multiple of 16 bytes
// are bound by instructions.  32768 x 2048: 59.6 us, 6.0 TB/s read and written.
constexpr int LOOK_NT = 256, LOOK_TX = 128;

template <int VEC, int U>  // U: columns per thread, loaded before the first is stored
__global__ void __launch_bounds__(LOOK_NT) k_embed(const float* __restrict__ table, int64_t ld,
                                                  const void* __restrict__ ids, int kind, int64_t n, int V,
                                                  uint32_t cols, int chunks, float scale, float* __restrict__ out,
                                                  int64_t ldo) {
  ::tp::pdl_enter();
  const uint32_t group = chunks == 1 ? blockIdx.x : blockIdx.x / (uint32_t)chunks, tx = blockDim.x;
  const int64_t i = (int64_t)group * blockDim.y + threadIdx.y;
  const uint32_t c0 = (blockIdx.x - group * chunks) * U * tx + threadIdx.x;
  if (i >= n || c0 >= cols) return;
  const uint32_t left = cols - c0;
  const int v = token_id(ids, kind, i);
  const bool in = v >= 0 && v < V;
  const float* src = table + v * ld + (int64_t)VEC * c0;
  float* dst = out + i * ldo + (int64_t)VEC * c0;
  Col<VEC> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) x[u] = in && u * tx < left ? Col<VEC>::load(src, u * tx) : Col<VEC>::zero().times(NAN);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u * tx < left) x[u].times(scale).store(dst, u * tx);
}

// Clears a row of D values by n threads, this one the t-th: 16-byte stores between
// its ends.
__device__ __forceinline__ void clear_row(float* row, int64_t D, int t, int n) {
  int64_t head = (4 - (((uintptr_t)row >> 2) & 3)) & 3;
  if (head > D) head = D;
  const int64_t body = (D - head) >> 2;
  if (t < head) row[t] = 0.0f;
  float4* mid = reinterpret_cast<float4*>(row + head);
#pragma unroll 4
  for (int64_t q = t; q < body; q += n) mid[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (t < D - head - 4 * body) row[head + 4 * body + t] = 0.0f;
}

// ---- gradient of a few tokens ---------------------------------------------------------
// One CTA per (position, 256 columns), which compares its token with all ids at
// once: the first position of a token sums all of them, in order.  Reads the ids
// n times over, and a frequent token's rows by one thread per column: 256 x 1024
// takes 5.2 us against 14.1 sorted, 1024 x 1024 7.2 against 16.9, but all of one
// token 77 against 16 (512 of them: 39), hence the bound.  Where rows are written,
// not added to, more CTAs clear `clear` rows each that no id names (2 x 2846 into
// 3946 rows: 7.8 us, 35 sorted).
constexpr int EMB_FEW = 512;
constexpr int FEW_U = 16;  // rows in flight (500 x 4096 of 10 tokens, added: 11.4 us, 14.4 with 8)
constexpr int FEW_CLEAR = 1024;       // rows that a CTA looks at, at most
constexpr int FEW_CLEAR_VALUES = 8192;  // values that it clears, if rows are shorter

template <int VEC, bool ACC>
__global__ void __launch_bounds__(256) k_embed_few(const float* __restrict__ dout, int64_t ldo,
                                                   const void* __restrict__ ids, int kind, int n, int64_t V,
                                                   int64_t cols, int chunks, float scale, int64_t pad,
                                                   float* __restrict__ dtable, int64_t ld, int clear) {
  ::tp::pdl_enter();
  if (!ACC && blockIdx.x >= (unsigned)n * chunks) {
    __shared__ bool present[FEW_CLEAR];
    const int t = threadIdx.x;
    const int64_t v0 = (int64_t)(blockIdx.x - (unsigned)n * chunks) * clear, D = cols * VEC;
    const int rows = (int)(V - v0 < clear ? V - v0 : clear);
    for (int r = t; r < rows; r += 256) present[r] = false;
    __syncthreads();
    for (int i = t; i < n; i += 256) {
      const int v = token_id(ids, kind, i);
      if (v >= v0 && v < v0 + rows && v != pad) present[v - v0] = true;
    }
    __syncthreads();
    float* first = dtable + v0 * ld;
    if (D < 32) {
      for (int e = t; e < rows * (int)D; e += 256) {
        const int r = e / (int)D;
        if (!present[r]) first[r * ld + e - r * (int)D] = 0.0f;
      }
    } else if (clear >= 8) {  // a warp per row
      for (int r = t >> 5; r < rows; r += 8)
        if (!present[r]) clear_row(first + r * ld, D, t & 31, 32);
    } else {
      for (int r = 0; r < rows; ++r)
        if (!present[r]) clear_row(first + r * ld, D, t, 256);
    }
    return;
  }
  __shared__ uint32_t hits[EMB_FEW / 32];
  __shared__ uint16_t list[EMB_FEW];
  const int t = threadIdx.x, lane = t & 31;
  const int i = blockIdx.x / chunks;
  const int64_t c = (int64_t)(blockIdx.x - i * chunks) * 256 + t;
  const int v = token_id(ids, kind, i);
  int u[EMB_FEW / 256];
#pragma unroll
  for (int r = 0; r < EMB_FEW / 256; ++r) u[r] = r * 256 + t < n ? token_id(ids, kind, r * 256 + t) : -1;
  if (v < 0 || v >= V || v == pad) return;
  bool earlier = false;
#pragma unroll
  for (int r = 0; r < EMB_FEW / 256; ++r) {
    earlier |= u[r] == v && r * 256 + t < i;
    const uint32_t b = __ballot_sync(0xffffffffu, u[r] == v);
    if (lane == 0) hits[r * 8 + (t >> 5)] = b;
  }
  if (__syncthreads_or(earlier)) return;
  int many = 0;  // the token's positions, in order
#pragma unroll
  for (int r = 0; r < EMB_FEW / 256; ++r) {
    int at = many;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const int k = __popc(hits[r * 8 + w]);
      at += w < t >> 5 ? k : 0;
      many += k;
    }
    if (u[r] == v) list[at + __popc(hits[r * 8 + (t >> 5)] & ((1u << lane) - 1))] = (uint16_t)(r * 256 + t);
  }
  __syncthreads();
  if (c >= cols) return;
  Col<VEC> old;
  if (ACC) old = Col<VEC>::load(dtable + (int64_t)v * ld, c);
  Col<VEC> acc = Col<VEC>::zero();
  const float* at = dout + (int64_t)VEC * c;
  int h = 0;
  for (; h + FEW_U <= many; h += FEW_U) {  // sums of FEW_U rows, then of these
    Col<VEC> x[FEW_U];
#pragma unroll
    for (int k = 0; k < FEW_U; ++k) x[k] = Col<VEC>::load(at + list[h + k] * ldo, 0);
#pragma unroll
    for (int k = 1; k < FEW_U; ++k) x[0].add(x[k]);
    acc.add(x[0]);
  }
#pragma unroll 4
  for (; h < many; ++h) acc.add(Col<VEC>::load(at + list[h] * ldo, 0));
  Col<VEC> r = acc.times(scale);
  if (ACC) r.add(old);
  r.store(dtable + (int64_t)v * ld, c);
}

// ---- gradient of many tokens: positions sorted by token, then summed -----------------------
// Sorting is one launch of G = 2^g CTAs that share nothing.  Token v belongs to
// CTA v mod G, as its token v / G (neighbouring ids, of like frequency, go to
// different CTAs).  Each CTA reads all ids: it counts those of the CTAs before
// it, which is where its own begin, and the tokens of its own per warp; after a
// scan over (token, warp) the warps place their positions in order.  A position
// and its token are written per valid id, the start of each token's run per
// token.  (Reading all ids G times is n G 4 bytes from L2; the rows they stand for
// are n D 4 bytes from HBM.)
constexpr int SORT_NT = 1024;
constexpr int SORT_WARPS = SORT_NT / 32;
constexpr int EMB_SMS = 148;              // of a B200: a workspace's size is asked for without a device too
constexpr int LEAST_G = 7, MOST_G = 10;   // log2 of the CTAs: 128 for its SMs, or more
constexpr int SORT_TOKENS = 1024;         // tokens of one CTA, at most (a thread each in the scan)
constexpr int SORT_WORDS = 1024;          // positions / 32 of one launch: their hits are kept in shared memory
constexpr int64_t SORT_READS = (int64_t)1 << 22;  // ids that the CTAs of one launch read in all, at most
static_assert((SORT_READS >> LEAST_G) <= 32 * SORT_WORDS, "more positions than hits are kept of");
static_assert(32 * SORT_WORDS <= 65536, "a list holds offsets of 16 bits");
constexpr int SORT_LIST = 768;            // hits that a warp lists before it places them
constexpr int PLACE_U = 4;                // ids of a thread in flight as an owner places its own
constexpr int SORT_U = 16;                // ids of a thread in flight, and words listed at once

struct EmbedSort {
  int g;          // log2 of the CTAs
  int per;        // tokens of one CTA, W
  int64_t n;
  int V, pad;
  const void* ids;
  int32_t* start;  // [G W + 1]: where the run of key owner * W + local starts; the last: how many positions there are
  int32_t* pos;    // [n]
  int32_t* tok;    // [n]
  __device__ __forceinline__ bool valid(int v) const { return (uint32_t)v < (uint32_t)V && v != pad; }
  __device__ __forceinline__ int owner(int v) const { return v & ((1 << g) - 1); }
  __device__ __forceinline__ int local(int v) const { return v >> g; }
  __device__ __forceinline__ int key(int v) const { return owner(v) * per + local(v); }
  __device__ __forceinline__ int total() const { return start[(int64_t)per << g]; }
};

// The counts [warps][W] of CTA `me`'s tokens l0 .. l0 + W - 1 become the places of
// each warp's positions, those of the first token starting at `base`; start[] is
// written.  Returns where the last token's end.
__device__ __forceinline__ int embed_places(const EmbedSort& e, int32_t* count, int me, int l0, int W, int base,
                                            int32_t* sh) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  int k[SORT_WARPS], c = 0;  // one thread per token
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
  int first = base + incl - c, end = base;
  for (int i = 0; i < w; ++i) first += sh[i];
  for (int i = 0; i < SORT_WARPS; ++i) end += sh[i];
  if (t < W) {
    e.start[(int64_t)me * e.per + l0 + t] = first;
    int at = first;
#pragma unroll
    for (int i = 0; i < SORT_WARPS; ++i) {
      count[i * W + t] = at;
      at += k[i];
    }
    if (me == (1 << e.g) - 1 && l0 + t == e.per - 1) e.start[(int64_t)e.per << e.g] = first + c;
  }
  __syncthreads();
  return end;
}

// Where this lane's key stands: its place among the lanes of `some` (the ones that
// call) with the same key, after the key's counter, which moves on by their number.
__device__ __forceinline__ int embed_take(uint32_t some, int key, int32_t* counter) {
  const int lane = threadIdx.x & 31;
  const uint32_t peers = __match_any_sync(some, key);
  const int rank = __popc(peers & ((1u << lane) - 1)), to = *counter;
  __syncwarp(some);
  if (rank == 0) *counter = to + __popc(peers);
  return to + rank;
}

template <int KIND>
__global__ void __launch_bounds__(SORT_NT) k_embed_sort(const EmbedSort e) {
  ::tp::pdl_enter();
  extern __shared__ int32_t sort_sm[];
  __shared__ int32_t sh[SORT_WARPS];
  const int W = e.per, me = blockIdx.x, t = threadIdx.x, lane = t & 31, w = t >> 5;
  int32_t* count = sort_sm;                                  // [warps][W]
  uint16_t* hits = (uint16_t*)(sort_sm + SORT_WARPS * W);    // [warps][SORT_LIST]
  uint32_t* words = (uint32_t*)(hits + SORT_WARPS * SORT_LIST);   // hits of 32 positions each
  const int n = (int)e.n, nwords = (n + 31) >> 5;  // at most SORT_WORDS
  const int per = (nwords + SORT_WARPS - 1) / SORT_WARPS;  // words of one warp: neighbours, so that order is kept
  const int w0 = per * w < nwords ? per * w : nwords, w1 = w0 + per < nwords ? w0 + per : nwords;
  for (int i = t; i < SORT_WARPS * W; i += SORT_NT) count[i] = 0;
  __syncthreads();
  auto token = [&](int word) {
    const int p = word * 32 + lane;
    return word < w1 && p < n ? token_id(e.ids, KIND, p) : -1;
  };
  int less = 0;
  for (int i = w0; i < w1; i += SORT_U) {
    int v[SORT_U];
    uint32_t mine = 0u;
    if (i + SORT_U <= w1 && (i + SORT_U) * 32 <= n) {
      const int32_t* at = static_cast<const int32_t*>(e.ids) + i * 32 + lane;  // either storage is 4 bytes
#pragma unroll
      for (int q = 0; q < SORT_U; ++q) v[q] = token_id(at + 32 * q, KIND, 0);
    } else {
#pragma unroll
      for (int q = 0; q < SORT_U; ++q) v[q] = token(i + q);
    }
#pragma unroll
    for (int q = 0; q < SORT_U; ++q) {
      const bool ok = e.valid(v[q]), hit = ok && e.owner(v[q]) == me;
      less += ok && e.owner(v[q]) < me;
      const uint32_t b = __ballot_sync(0xffffffffu, hit);
      if (hit) atomicAdd(&count[w * W + e.local(v[q])], 1);
      mine = lane == q ? b : mine;
    }
    if (lane < SORT_U && i + lane < w1) words[i + lane] = mine;
  }
  for (int o = 16; o > 0; o >>= 1) less += __shfl_xor_sync(0xffffffffu, less, o);
  if (lane == 0) sh[w] = less;
  __syncthreads();
  int base = 0;
  for (int i = 0; i < SORT_WARPS; ++i) base += sh[i];
  __syncthreads();
  embed_places(e, count, me, 0, W, base, sh);
  // 16 words at a time, a lane lists its word's hits, in order, as offsets from the
  // list's first word; a list that has grown long is placed, 32 hits at a time, a
  // lane each, the tokens of the next 32 under way.
  uint16_t* list = hits + SORT_LIST * w;
  int have = 0;
  int list0 = w0;  // the word that offsets count from
  for (int i = w0; i < w1; i += SORT_U) {
    uint32_t mine = lane < SORT_U && i + lane < w1 ? words[i + lane] : 0u;
    int at = __popc(mine);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += u;
    }
    const int more = __shfl_sync(0xffffffffu, at, 31);
    at += have - __popc(mine);
    for (; mine; mine &= mine - 1) list[at++] = (uint16_t)(32 * (i - list0 + lane) + __ffs(mine) - 1);
    have += more;
    // room for 16 words more, or the end
    if (have <= SORT_LIST - 32 * SORT_U && i + SORT_U < w1) continue;
    __syncwarp();
    const int first = list0 * 32;
    auto fetch = [&](int h) { return h < have ? token_id(e.ids, KIND, first + list[h]) : 0; };
    int v = fetch(lane);
    for (int h = 0; h < have; h += 32) {
      const int next = fetch(h + 32 + lane), k = have - h < 32 ? have - h : 32;
      if (lane < k) {
        const int to = embed_take(k == 32 ? 0xffffffffu : (1u << k) - 1, v, &count[w * W + e.local(v)]);
        e.pos[to] = first + list[h + lane];
        e.tok[to] = v;
      }
      __syncwarp();
      v = next;
    }
    have = 0;
    list0 = i + SORT_U;
  }
}

// Of many ids, or of a vocabulary of more CTAs than SMs, reading all G times is too
// much.  They are then split by owner first: each of B CTAs counts the owners in its
// share of the positions; each, knowing all counts, moves its share to where it
// belongs, order kept; and G CTAs sort what is theirs by token, which is all they
// read.  (262144 ids of 32000 tokens: 28 us against 53.)  Owners of more tokens than
// a CTA sorts at once (a vocabulary above 2^20) go through theirs again for each
// SORT_TOKENS of them (262144 ids of 2 million tokens, 64 wide, added: 151 us; with
// 2048 owners that each read all ids 552; 16384 ids: 91 and 98).
struct EmbedSplit {
  int64_t share;     // words of a CTA
  int32_t* count;    // [B][G]
  int32_t* first;    // [G + 1]: where an owner's positions start
  int32_t* pos;      // [n], by owner
  int32_t* tok;      // [n]
};

template <int KIND>
__global__ void __launch_bounds__(SORT_NT) k_embed_count(const EmbedSort e, const EmbedSplit p) {
  ::tp::pdl_enter();
  __shared__ int32_t owners[1 << MOST_G];
  const int G = 1 << e.g;
  for (int i = threadIdx.x; i < G; i += SORT_NT) owners[i] = 0;
  __syncthreads();
  const int64_t from = blockIdx.x * p.share * 32, to = from + p.share * 32 < e.n ? from + p.share * 32 : e.n;
#pragma unroll 4
  for (int64_t i = from + threadIdx.x; i < to; i += SORT_NT) {
    const int v = token_id(e.ids, KIND, i);
    if (e.valid(v)) atomicAdd(&owners[e.owner(v)], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G; i += SORT_NT) p.count[(int64_t)blockIdx.x * G + i] = owners[i];
}

template <int KIND>
__global__ void __launch_bounds__(SORT_NT) k_embed_split(const EmbedSort e, const EmbedSplit p) {
  ::tp::pdl_enter();
  extern __shared__ int32_t sort_sm[];  // [warps][G]: counts, then places
  __shared__ int32_t all[1 << MOST_G], before[1 << MOST_G], sh[SORT_WARPS];
  const int G = 1 << e.g, t = threadIdx.x, lane = t & 31, w = t >> 5;
  for (int i = t; i < SORT_WARPS * G; i += SORT_NT) sort_sm[i] = 0;
  for (int i = t; i < G; i += SORT_NT) all[i] = before[i] = 0;
  __syncthreads();
  {  // of each owner: how many there are, and how many in the shares before this one
    const int o = t & (G - 1);
    int sum = 0, less = 0;
#pragma unroll 8
    for (int b = t >> e.g; b < (int)gridDim.x; b += SORT_NT >> e.g) {
      const int c = p.count[(int64_t)b * G + o];
      sum += c;
      less += b < (int)blockIdx.x ? c : 0;
    }
    atomicAdd(&all[o], sum);
    atomicAdd(&before[o], less);
  }
  const int64_t nwords = (e.n + 31) >> 5, from = blockIdx.x * p.share, to = from + p.share < nwords ? from + p.share : nwords;
  const int64_t per = (p.share + SORT_WARPS - 1) / SORT_WARPS;
  const int64_t w0 = from + per * w < to ? from + per * w : to, w1 = w0 + per < to ? w0 + per : to;
  int32_t* mine = sort_sm + w * G;
  auto token = [&](int64_t word) {
    const int64_t i = word * 32 + lane;
    const int v = i < e.n ? token_id(e.ids, KIND, i) : -1;
    return e.valid(v) ? v : -1;
  };
#pragma unroll 4
  for (int64_t i = w0; i < w1; ++i) {
    const int v = token(i);
    if (v >= 0) atomicAdd(&mine[e.owner(v)], 1);
  }
  __syncthreads();
  int incl = t < G ? all[t] : 0;  // scan over the owners
  const int own = incl;
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) sh[w] = incl;
  __syncthreads();
  int first = incl - own;
  for (int i = 0; i < w; ++i) first += sh[i];
  if (t < G) {
    if (blockIdx.x == 0) {
      p.first[t] = first;
      if (t == G - 1) p.first[G] = first + own;
    }
    int at = first + before[t];
    for (int i = 0; i < SORT_WARPS; ++i) {
      const int c = sort_sm[i * G + t];
      sort_sm[i * G + t] = at;
      at += c;
    }
  }
  __syncthreads();
  int next = w0 < w1 ? token(w0) : -1;
  for (int64_t i = w0; i < w1; ++i) {
    const int v = next;
    if (i + 1 < w1) next = token(i + 1);
    const uint32_t some = __ballot_sync(0xffffffffu, v >= 0);
    if (v >= 0) {
      const int to = embed_take(some, e.owner(v), &mine[e.owner(v)]);
      p.pos[to] = (int32_t)(i * 32 + lane);
      p.tok[to] = v;
    }
    __syncwarp();
  }
}

__global__ void __launch_bounds__(SORT_NT) k_embed_place(const EmbedSort e, const EmbedSplit p) {
  ::tp::pdl_enter();
  extern __shared__ int32_t sort_sm[];  // [warps][W], W tokens at once
  __shared__ int32_t sh[SORT_WARPS];
  const int me = blockIdx.x, t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int begin = p.first[me], end = p.first[me + 1];
  const int per = ((end - begin + SORT_NT - 1) / SORT_NT) * 32;  // of a warp
  const int64_t s0 = (int64_t)begin + (int64_t)per * w;
  const int64_t i0 = s0 < end ? s0 : end, i1 = i0 + per < end ? i0 + per : end;
  int base = begin;
  for (int l0 = 0; l0 < e.per; l0 += SORT_TOKENS) {
    const int W = e.per - l0 < SORT_TOKENS ? e.per - l0 : SORT_TOKENS;
    for (int i = t; i < SORT_WARPS * W; i += SORT_NT) sort_sm[i] = 0;
    __syncthreads();
    int32_t* mine = sort_sm + w * W;
    auto local = [&](int v) { return e.local(v) - l0; };
#pragma unroll 4
    for (int64_t i = i0 + lane; i < i1; i += 32) {
      const int l = local(p.tok[i]);
      if ((uint32_t)l < (uint32_t)W) atomicAdd(&mine[l], 1);
    }
    __syncthreads();
    base = embed_places(e, sort_sm, me, l0, W, base, sh);
    for (int64_t i = i0; i < i1; i += 32 * PLACE_U) {
      int v[PLACE_U], at[PLACE_U];
#pragma unroll
      for (int q = 0; q < PLACE_U; ++q) {
        const int64_t j = i + 32 * q + lane;
        v[q] = j < i1 ? p.tok[j] : -1;
        at[q] = j < i1 ? p.pos[j] : 0;
      }
#pragma unroll
      for (int q = 0; q < PLACE_U; ++q) {
        const bool take = v[q] >= 0 && (uint32_t)local(v[q]) < (uint32_t)W;
        const uint32_t some = __ballot_sync(0xffffffffu, take);
        if (take) {
          const int to = embed_take(some, v[q], &mine[local(v[q])]);
          e.pos[to] = at[q];
          e.tok[to] = v[q];
        }
        __syncwarp();
      }
    }
    __syncthreads();
  }
}

// Tiles of T sorted positions are summed each by itself, so a frequent token
// takes no longer than many rare ones.  A run (the positions of one token) of at
// most 2 T goes whole to the tile it starts in.  A longer one is cut at the
// tiles' borders: what came in from the tile before is the tile's partial 0, the
// start of what goes on its partial 1 (what does both, partial 0).  T is 64, or 32
// or 16 where 64 would leave SMs without a tile (added: 65536 x 1024 98 us with 64,
// 105 with 24; 4096 x 4096 39.3, 42.6 with 16; 4147 x 3243 39.0 with 32, 42.3 with 16).
// 16384 x 4096 into 32000 rows written whole: 119 us, 6.6 TB/s.
struct EmbedSum {
  const float* dout;
  int64_t ldo, cols;
  int chunks, T;
  int64_t tiles, tile_ctas;
  float scale;
  float* dtable;
  int64_t ld;
  float* partial;  // [2 tiles][ldp]
  int64_t ldp;
  int2* cut;       // [tiles]: the cut run that starts in a tile: its token (-1: none) and its last tile
};

constexpr int SUM_U = 8;     // rows in flight per thread (two 16-byte vectors of positions)
constexpr int SUM_ZERO = 4;  // rows looked at by a warp (or thread) that clears those of absent tokens

template <int VEC>
__device__ __forceinline__ void embed_zero(const EmbedSort& e, const EmbedSum& a, int64_t group) {
  if (blockDim.x < 32) {  // narrow rows: a thread per column
    const int64_t v0 = (group * blockDim.y + threadIdx.y) * SUM_ZERO;
    if (threadIdx.x >= a.cols) return;
    for (int64_t v = v0; v < v0 + SUM_ZERO && v < e.V; ++v) {
      const int k = e.key((int)v);
      if (e.start[k] == e.start[k + 1]) Col<VEC>::zero().store(a.dtable + v * a.ld, threadIdx.x);
    }
    return;
  }
  // a warp per row, in 16-byte stores between its ends
  const int t = threadIdx.y * blockDim.x + threadIdx.x, lane = t & 31;
  const int64_t v0 = (group * (EMB_NT / 32) + (t >> 5)) * SUM_ZERO, D = a.cols * VEC;
  bool gone = false;
  if (lane < SUM_ZERO && v0 + lane < e.V) {
    const int k = e.key((int)(v0 + lane));
    gone = e.start[k] == e.start[k + 1];
  }
  for (uint32_t some = __ballot_sync(0xffffffffu, gone); some; some &= some - 1)
    clear_row(a.dtable + (v0 + __ffs(some) - 1) * a.ld, D, lane, 32);
}

// (4 CTAs to an SM with the old values in flight, at 128 registers and 24 bytes
// spilled: its registers would leave 3, and 131622 x 332 added then takes 94.5 us
// instead of 87.4; 8 CTAs would spill 920.)
template <int VEC, bool ACC>
__global__ void __launch_bounds__(EMB_NT, VEC == 4 && ACC ? 4 : 1) k_embed_sum(const EmbedSort e, const EmbedSum a) {
  ::tp::pdl_enter();
  if (blockIdx.x >= a.tile_ctas * a.chunks) {
    embed_zero<VEC>(e, a, blockIdx.x - a.tile_ctas * a.chunks);
    return;
  }
  const int64_t group = blockIdx.x / a.chunks;
  const int64_t c = (int64_t)(blockIdx.x - group * a.chunks) * blockDim.x + threadIdx.x;
  const int64_t tile = group * blockDim.y + threadIdx.y;
  if (c >= a.cols || tile >= a.tiles) return;
  const int T = a.T, m = e.total();
  int2 starts = make_int2(-1, 0);
  if (tile * T >= m) {
    if (c == 0) a.cut[tile] = starts;
    return;
  }
  const int s0 = (int)(tile * T);
  int s1 = m - s0 < T ? m : s0 + T, from = s0;
  const int first = e.tok[s0], before = s0 > 0 ? e.tok[s0 - 1] : -1;
  const int final = e.tok[s1 - 1], after = s1 < m ? e.tok[s1] : -1;
  bool came_in = false, goes_on = false;
  if (before == first) {
    const int k = e.key(first), end = e.start[k + 1];
    if (end - e.start[k] > 2 * T) came_in = true;
    else from = end;
  }
  if (after == final) {
    const int k = e.key(final), start = e.start[k], end = e.start[k + 1];
    if (end - start > 2 * T) {
      goes_on = true;
      if (start >= s0) starts = make_int2(final, (end - 1) / T);
    } else if (start >= s0) {
      s1 = end;
    }
  }
  if (c == 0) a.cut[tile] = starts;
  if (from >= s1) return;  // all of it belongs to a run of the tile before
  int cur = e.tok[from];
  float* part = a.partial + 2 * tile * a.ldp;
  Col<VEC> acc = Col<VEC>::zero();
  auto flush = [&](const Col<VEC>& old) {
    if (came_in) {
      acc.store(part, c);
    } else {
      Col<VEC> r = acc.times(a.scale);
      if (ACC) r.add(old);
      r.store(a.dtable + (int64_t)cur * a.ld, c);
    }
  };
  // eight positions at a time, on eight-position boundaries (one past the last is
  // still inside the workspace), those of the next batch fetched ahead (65536 x 1024
  // added: 98 us, 104 without); lo, hi: which of them are the tile's
  int4 nt0, nt1, np0, np1;
  auto fetch = [&](int s) {
    nt0 = *reinterpret_cast<const int4*>(e.tok + s), nt1 = *reinterpret_cast<const int4*>(e.tok + s + 4);
    np0 = *reinterpret_cast<const int4*>(e.pos + s), np1 = *reinterpret_cast<const int4*>(e.pos + s + 4);
  };
  auto batch = [&](int s, int lo, int hi) {
    const int4 t0 = nt0, t1 = nt1, p0 = np0, p1 = np1;
    if (s + SUM_U < s1) fetch(s + SUM_U);
    const int tok[SUM_U] = {t0.x, t0.y, t0.z, t0.w, t1.x, t1.y, t1.z, t1.w};
    const int pos[SUM_U] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
    Col<VEC> x[SUM_U], old[ACC ? SUM_U : 1];
#pragma unroll
    for (int k = 0; k < SUM_U; ++k)
      if (k >= lo && k < hi) x[k] = Col<VEC>::load(a.dout + (int64_t)pos[k] * a.ldo, c);
    if (ACC)  // the rows that runs ending in this batch are added to (each is this thread's alone)
#pragma unroll
      for (int k = 0; k < SUM_U; ++k)
        if (k >= lo && k < hi) {
          const int prev = k > lo ? tok[k > 0 ? k - 1 : 0] : cur;
          if (tok[k] != prev) old[k] = Col<VEC>::load(a.dtable + (int64_t)prev * a.ld, c);
        }
#pragma unroll
    for (int k = 0; k < SUM_U; ++k)
      if (k >= lo && k < hi) {
        if (tok[k] != cur) {
          flush(old[ACC ? k : 0]);
          cur = tok[k];
          came_in = false;
          acc = Col<VEC>::zero();
        }
        acc.add(x[k]);
      }
  };
  int s = from & ~(SUM_U - 1);
  fetch(s);
  if (s < from) {
    batch(s, from - s, s1 - s < SUM_U ? s1 - s : SUM_U);
    s += SUM_U;
  }
  for (; s + SUM_U <= s1; s += SUM_U) batch(s, 0, SUM_U);
  if (s < s1) batch(s, 0, s1 - s);
  if (!came_in && goes_on) {
    acc.store(part + a.ldp, c);
  } else {
    Col<VEC> old;
    if (ACC && !came_in) old = Col<VEC>::load(a.dtable + (int64_t)cur * a.ld, c);
    flush(old);
  }
}

// The runs that were cut: the tile one starts in adds up its partial 1 and the
// partials 0 of the tiles after it, in f64: a CTA is `across` threads wide, its
// rows of threads take every so many-th tile, and their sums meet pair by pair.  A
// CTA looks through 8 tiles for such starts (16384 x 4096: 7 us; through 32: 11).
constexpr int JOIN_TILES = 8, JOIN_NT = 256;

template <bool ACC>
__global__ void __launch_bounds__(JOIN_NT) k_embed_join(const EmbedSum a, int64_t D, int chunks, int across) {
  ::tp::pdl_enter();
  __shared__ double sh[4][JOIN_NT];
  const int t = threadIdx.x, lane = t & 31, r = t / across, rows = JOIN_NT / across;
  const int64_t group = blockIdx.x / chunks;
  const int64_t c4 = (int64_t)(blockIdx.x - group * chunks) * across + t - r * across;  // a 4-value column of the partials
  const int64_t mine = group * JOIN_TILES + lane;                                 // every warp looks at the same tiles
  const int2 run = lane < JOIN_TILES && mine < a.tiles ? a.cut[mine] : make_int2(-1, 0);
  for (uint32_t some = __ballot_sync(0xffffffffu, run.x >= 0); some; some &= some - 1) {
    const int which = __ffs(some) - 1;
    const int64_t tile = group * JOIN_TILES + which;
    const int v = __shfl_sync(0xffffffffu, run.x, which), last = __shfl_sync(0xffffffffu, run.y, which);
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    auto add = [&](int64_t row) {
      const float4 x = *(reinterpret_cast<const float4*>(a.partial + row * a.ldp) + c4);
      acc[0] += x.x;
      acc[1] += x.y;
      acc[2] += x.z;
      acc[3] += x.w;
    };
    if (4 * c4 < D) {
      if (r == 0) add(2 * tile + 1);
#pragma unroll 8
      for (int64_t k = tile + 1 + r; k <= last; k += rows) add(2 * k);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) sh[q][t] = acc[q];
    __syncthreads();
    int o = rows / 2;
    while (o >= last - tile) o >>= 1;  // rows from last - tile on have nothing
    for (; o > 0; o >>= 1) {
      if (r < o)
#pragma unroll
        for (int q = 0; q < 4; ++q) sh[q][t] += sh[q][t + o * across];
      __syncthreads();
    }
    if (r == 0) {
      float* row = a.dtable + (int64_t)v * a.ld + 4 * c4;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (4 * c4 + q < D) {
          const float g = (float)(sh[q][t] * a.scale);
          row[q] = ACC ? row[q] + g : g;
        }
    }
    __syncthreads();
  }
}

// ---- launches -----------------------------------------------------------------------------
// the widest column that D and the rows of both buffers allow
static int col_width(int64_t D, const void* p, int64_t ldp, const void* q, int64_t ldq) {
  const int64_t all = D | ldp | ldq | (int64_t)((((uintptr_t)p | (uintptr_t)q) & 15) >> 2);
  return all % 4 == 0 ? 4 : (all % 2 == 0 ? 2 : 1);
}

static unsigned grid_of(int64_t groups, int64_t chunks, const char* what) {
  TP_REQUIRE(groups <= INT_MAX / chunks, "%s: too many tokens, rows or columns for one launch", what);
  return (unsigned)(groups * chunks);
}

void launch_embed(const float* table, int64_t ld, const void* ids, int kind, int64_t n, int64_t V, int64_t D,
                  float scale, float* out, int64_t ldo) {
  if (n == 0 || D == 0) return;
  const int vec = col_width(D, table, ld, out, ldo);
  const int64_t cols = D / vec;
  // columns of a thread; 20000 x 777 by 16 17.5 us, by 8 21.2; 200000 x 33 14.3 and 10.7
  const int U = vec == 4 ? 4 : (vec == 1 && cols > 512 ? 16 : 8);
  const int64_t need = (cols + U - 1) / U;  // threads
  const int chunks = (int)((need + LOOK_TX - 1) / LOOK_TX);
  int tx = block_cols(need);
  if (tx > 32) tx = (int)(((need + chunks - 1) / chunks + 31) / 32 * 32);
  const int ty = LOOK_NT / tx;
  const unsigned grid = grid_of((n + ty - 1) / ty, chunks, "token_embedding");
#define TP_EMBED(VEC, U)                                                                                         \
  TP_LAUNCH((k_embed<VEC, U>), grid, dim3(tx, ty), 0, table, ld, ids, kind, n, (int)V, (uint32_t)cols, chunks, scale, \
            out, ldo)
  if (vec == 4) TP_EMBED(4, 4);
  else if (vec == 2) TP_EMBED(2, 8);
  else if (U == 16) TP_EMBED(1, 16);
  else TP_EMBED(1, 8);
#undef TP_EMBED
}

struct EmbedPlan {
  int64_t per, start, pos, tok, cut, count, first, spos, stok, partial, ldp, bytes, tiles, share;
  int g, T, B;
  bool split;
  EmbedPlan(int64_t n, int64_t V, int64_t D) {  // n > 0
    g = LEAST_G;
    while (g < MOST_G && ((int64_t)SORT_TOKENS << g) < V) ++g;
    per = (V + (1 << g) - 1) >> g;
    const int64_t work = n / 64 * D / 512;  // CTAs of 512 columns by 64 positions
    T = work >= EMB_SMS * 4 ? 64 : (work >= EMB_SMS * 2 ? 32 : 16);
    tiles = (n + T - 1) / T;
    ldp = (D + 3) / 4 * 4;
    auto up = [](int64_t b) { return (b + 15) / 16 * 16; };
    start = 0;
    pos = start + up(((per << g) + 1) * 4);
    tok = pos + up(n * 4 + 32);
    cut = tok + up(n * 4 + 32);
    // the whole gradient at a width of 64: 32768 ids of 32000 tokens 24.8 us in one
    // launch, 27.5 split first; 65536 ids 33.9 and 31.6
    split = per > SORT_TOKENS || n << g > SORT_READS;
    const int64_t words = (n + 31) / 32;
    share = (words + EMB_SMS - 1) / EMB_SMS;
    B = split ? (int)((words + share - 1) / share) : 0;
    count = cut + up(tiles * 8);
    first = count + up((int64_t)B * 4 << g);
    spos = first + (split ? up(4 + (4 << g)) : 0);
    stok = spos + (split ? up(n * 4) : 0);
    partial = stok + (split ? up(n * 4) : 0);
    bytes = partial + 2 * tiles * ldp * 4;
  }
};

int64_t embed_bwd_ws(int64_t n, int64_t V, int64_t D) { return n <= EMB_FEW ? 0 : EmbedPlan(n, V, D).bytes; }

template <int VEC, bool ACC>
static void launch_sum(const EmbedSort& e, EmbedSum a, int64_t D) {
  const char* what = "token_embedding_backward";
  a.cols = D / VEC;
  const int tx = block_cols(a.cols), ty = EMB_NT / tx;
  a.chunks = (int)((a.cols + tx - 1) / tx);
  a.tile_ctas = (a.tiles + ty - 1) / ty;
  const int64_t rows = (tx < 32 ? ty : EMB_NT / 32) * SUM_ZERO;  // of one clearing CTA
  const int64_t zero_ctas = ACC ? 0 : (e.V + rows - 1) / rows;
  const int64_t grid = (int64_t)grid_of(a.tile_ctas, a.chunks, what) + zero_ctas;
  TP_REQUIRE(grid <= INT_MAX, "%s: too many tokens, rows or columns for one launch", what);
  TP_LAUNCH((k_embed_sum<VEC, ACC>), (unsigned)grid, dim3(tx, ty), 0, e, a);
  int across = 1;
  while (across < 32 && 4 * across < D) across *= 2;
  const int jchunks = (int)((D + 4 * across - 1) / (4 * across));
  TP_LAUNCH(k_embed_join<ACC>, grid_of((a.tiles + JOIN_TILES - 1) / JOIN_TILES, jchunks, what), JOIN_NT, 0, a, D,
            jchunks, across);
}

// Lets a kernel have that much dynamic shared memory; asked for once per kernel.
template <class K>
static void raise_smem(K* kernel, int bytes) {
  static std::vector<void*> done;
  for (void* k : done)
    if (k == (void*)kernel) return;
  TP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.push_back((void*)kernel);
}

void launch_embed_bwd(const float* dout, int64_t ldo, const void* ids, int kind, int64_t n, int64_t V, int64_t D,
                      float scale, int64_t pad, bool accumulate, float* dtable, int64_t ld, void* ws) {
  if (D == 0 || (n == 0 && accumulate)) return;
  const int vec = col_width(D, dout, ldo, dtable, ld);
  if (n <= EMB_FEW) {
    const char* what = "token_embedding_backward";
    const int64_t cols = D / vec;
    const int chunks = (int)((cols + 255) / 256);
    const int clear = (int)(FEW_CLEAR_VALUES / D < 1 ? 1 : (FEW_CLEAR_VALUES / D < FEW_CLEAR ? FEW_CLEAR_VALUES / D : FEW_CLEAR));
    const int64_t grid = (int64_t)grid_of(n, chunks, what) + (accumulate ? 0 : (V + clear - 1) / clear);
    TP_REQUIRE(grid <= INT_MAX, "%s: too many tokens, rows or columns for one launch", what);
#define TP_FEW(VEC, ACC)                                                                                          \
  TP_LAUNCH((k_embed_few<VEC, ACC>), (unsigned)grid, 256, 0, dout, ldo, ids, kind, (int)n, V, cols, chunks, scale, pad, \
            dtable, ld, clear)
    if (accumulate && vec == 4) TP_FEW(4, true);
    else if (accumulate && vec == 2) TP_FEW(2, true);
    else if (accumulate) TP_FEW(1, true);
    else if (vec == 4) TP_FEW(4, false);
    else if (vec == 2) TP_FEW(2, false);
    else TP_FEW(1, false);
#undef TP_FEW
    return;
  }
  const EmbedPlan p(n, V, D);
  char* base = (char*)ws;
  EmbedSort e;
  e.g = p.g;
  e.per = (int)p.per;
  e.n = n;
  e.V = (int)V;
  e.pad = (int)pad;
  e.ids = ids;
  e.start = (int32_t*)(base + p.start);
  e.pos = (int32_t*)(base + p.pos);
  e.tok = (int32_t*)(base + p.tok);
  const bool i32 = kind == IDS_I32;
  if (p.split) {
    EmbedSplit s;
    s.share = p.share;
    s.count = (int32_t*)(base + p.count);
    s.first = (int32_t*)(base + p.first);
    s.pos = (int32_t*)(base + p.spos);
    s.tok = (int32_t*)(base + p.stok);
    raise_smem(k_embed_split<IDS_I32>, SORT_WARPS * 4 << MOST_G);
    raise_smem(k_embed_split<IDS_F32>, SORT_WARPS * 4 << MOST_G);
    raise_smem(k_embed_place, SORT_WARPS * 4 * SORT_TOKENS);
    TP_LAUNCH(i32 ? k_embed_count<IDS_I32> : k_embed_count<IDS_F32>, p.B, SORT_NT, 0, e, s);
    TP_LAUNCH(i32 ? k_embed_split<IDS_I32> : k_embed_split<IDS_F32>, p.B, SORT_NT, (size_t)SORT_WARPS * 4 << p.g, e, s);
    const int64_t W = p.per < SORT_TOKENS ? p.per : SORT_TOKENS;
    TP_LAUNCH(k_embed_place, 1u << p.g, SORT_NT, (size_t)SORT_WARPS * 4 * W, e, s);
  } else {
    // at most 128 KB of counts, 48 of listed hits, 4 of hits
    const int most = (SORT_WARPS * (SORT_TOKENS + SORT_LIST / 2) + SORT_WORDS) * 4;
    const int64_t words = (n + 31) / 32;
    const size_t smem = (size_t)(SORT_WARPS * (p.per + SORT_LIST / 2) + words) * 4;
    raise_smem(k_embed_sort<IDS_I32>, most);
    raise_smem(k_embed_sort<IDS_F32>, most);
    TP_LAUNCH(i32 ? k_embed_sort<IDS_I32> : k_embed_sort<IDS_F32>, 1u << p.g, SORT_NT, smem, e);
  }
  EmbedSum a;
  a.dout = dout;
  a.ldo = ldo;
  a.T = p.T;
  a.tiles = p.tiles;
  a.scale = scale;
  a.dtable = dtable;
  a.ld = ld;
  a.partial = (float*)(base + p.partial);
  a.ldp = p.ldp;
  a.cut = (int2*)(base + p.cut);
  if (accumulate && vec == 4) launch_sum<4, true>(e, a, D);
  else if (accumulate && vec == 2) launch_sum<2, true>(e, a, D);
  else if (accumulate) launch_sum<1, true>(e, a, D);
  else if (vec == 4) launch_sum<4, false>(e, a, D);
  else if (vec == 2) launch_sum<2, false>(e, a, D);
  else launch_sum<1, false>(e, a, D);
}

// Most positions: the gradient's kernels round them up to SORT_NT (a share of a
// warp) and to SUM_U (a batch) in 32 bits.
constexpr int64_t LOOK_MOST = INT_MAX - 1, EMB_MOST = ((int64_t)1 << 31) - 2048;
static_assert(EMB_MOST + SORT_NT <= INT_MAX && EMB_MOST + SUM_U <= INT_MAX, "positions are rounded up in 32 bits");

static void check_embed(int64_t n, int64_t most, int64_t V, int64_t D, int64_t ld, int64_t ldo, const char* what) {
  TP_REQUIRE(n >= 0 && n <= most, "%s: %lld tokens is outside [0, %lld]", what, (long long)n, (long long)most);
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
    check_embed(n, LOOK_MOST, vocab, dim, ld, ldo, what);
    check_ids_kind(ids_kind, what);
    if (n == 0 || dim == 0) return;
    TP_REQUIRE(table && ids && out, "%s: table, ids and out must not be NULL", what);
    check_aligned({table, ids, out}, what);
    TP_REQUIRE(out != table && (const void*)out != ids, "%s: out is an input", what);
    launch_embed(table, ld, ids, ids_kind, n, vocab, dim, scale, out, ldo);
  });
}

TP_API int tpk_token_embedding_backward_ws(int64_t n, int64_t vocab, int64_t dim, int64_t* bytes) {
  return guard([&] {
    check_embed(n, EMB_MOST, vocab, dim, dim, dim, "token_embedding_backward_ws");
    TP_REQUIRE(bytes, "token_embedding_backward_ws: bytes is NULL");
    *bytes = embed_bwd_ws(n, vocab, dim);
  });
}

TP_API int tpk_token_embedding_backward(const float* dout, int64_t ldo, const void* ids, int ids_kind, int64_t n,
                                        int64_t vocab, int64_t dim, float scale, int64_t padding_id, int accumulate,
                                        float* dtable, int64_t ld, void* ws, int64_t ws_bytes) {
  return guard([&] {
    const char* what = "token_embedding_backward";
    check_embed(n, EMB_MOST, vocab, dim, ld, ldo, what);
    check_ids_kind(ids_kind, what);
    TP_REQUIRE(padding_id >= -1 && padding_id < vocab, "%s: padding_id %lld is neither -1 nor a row of the table",
               what, (long long)padding_id);
    TP_REQUIRE(accumulate == 0 || accumulate == 1, "%s: accumulate must be 0 or 1, got %d", what, accumulate);
    if (dim == 0) return;
    TP_REQUIRE(dtable && (n == 0 || (dout && ids)), "%s: dout, ids and dtable must not be NULL", what);
    check_aligned({dout, ids, dtable}, what);
    TP_REQUIRE(dtable != dout && (const void*)dtable != ids, "%s: dtable is an input", what);
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
    check_embed(I.numel, LOOK_MOST, T.shape[0], T.shape[1], T.shape[1], T.shape[1], what);
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
    check_embed(n, EMB_MOST, vocab, D, D, D, what);
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
