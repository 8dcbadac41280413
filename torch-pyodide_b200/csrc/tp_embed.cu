// Rows of a table by token id, scaled, and the table's gradient.
//
//   out_i = scale * table[id_i]         dtable_v (+)= scale * sum over { i : id_i = v } of dout_i
//
// The sum runs in an order fixed by the positions alone (no float atomics), so
// equal inputs give equal bits.
#include <cuda_runtime.h>

#include <climits>

#include "tp_core.h"
#include "tp_launch.h"
#include "tp_token.cuh"

namespace tp {

__global__ void __launch_bounds__(256) k_embed(const float* table, int64_t ld, const void* ids, int kind, int64_t n,
                                               int64_t V, int64_t D, float scale, float* out, int64_t ldo) {
  ::tp::pdl_enter();
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
    const int64_t v = token_id(ids, kind, i);
    const bool in = v >= 0 && v < V;
    for (int64_t d = threadIdx.x; d < D; d += 256) out[i * ldo + d] = in ? table[v * ld + d] * scale : NAN;
  }
}

// One CTA per (position, 256 columns): the first position of a token sums all
// of them, in order.
__global__ void __launch_bounds__(256) k_embed_bwd(const float* dout, int64_t ldo, const void* ids, int kind,
                                                   int64_t n, int64_t V, int64_t D, float scale, int64_t pad,
                                                   int accumulate, float* dtable, int64_t ld) {
  ::tp::pdl_enter();
  __shared__ uint32_t hit[8];
  const int64_t i = blockIdx.x, d = (int64_t)blockIdx.y * 256 + threadIdx.x;
  const int64_t v = token_id(ids, kind, i);
  if (v < 0 || v >= V || v == pad) return;
  bool earlier = false;
  for (int64_t j = threadIdx.x; j < i; j += 256) earlier |= token_id(ids, kind, j) == v;
  if (__syncthreads_or(earlier)) return;
  float acc = 0.0f;
  for (int64_t j0 = i; j0 < n; j0 += 256) {
    const int64_t j = j0 + threadIdx.x;
    const uint32_t b = __ballot_sync(0xffffffffu, j < n && token_id(ids, kind, j) == v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) hit[threadIdx.x >> 5] = b;
    __syncthreads();
    for (int w = 0; w < 8; ++w)
      for (uint32_t q = hit[w]; q; q &= q - 1)
        if (d < D) acc += dout[(j0 + 32 * w + __ffs(q) - 1) * ldo + d];
  }
  if (d < D) dtable[v * ld + d] = accumulate ? dtable[v * ld + d] + acc * scale : acc * scale;
}

void launch_embed(const float* table, int64_t ld, const void* ids, int kind, int64_t n, int64_t V, int64_t D,
                  float scale, float* out, int64_t ldo) {
  if (n == 0 || D == 0) return;
  TP_LAUNCH(k_embed, (unsigned)(n < 65536 ? n : 65536), 256, 0, table, ld, ids, kind, n, V, D, scale, out, ldo);
}

int64_t embed_bwd_ws(int64_t n, int64_t V, int64_t D) { return 16; }

void launch_embed_bwd(const float* dout, int64_t ldo, const void* ids, int kind, int64_t n, int64_t V, int64_t D,
                      float scale, int64_t pad, bool accumulate, float* dtable, int64_t ld, void* ws) {
  if (!accumulate)
    TP_CUDA(cudaMemset2DAsync(dtable, (size_t)ld * 4, 0, (size_t)D * 4, (size_t)V, stream()));
  if (n == 0 || D == 0) return;
  TP_LAUNCH(k_embed_bwd, dim3((unsigned)n, (unsigned)((D + 255) / 256)), 256, 0, dout, ldo, ids, kind, n, V, D, scale,
            pad, accumulate ? 1 : 0, dtable, ld);
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
