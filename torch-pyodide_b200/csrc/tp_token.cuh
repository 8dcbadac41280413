// What the entries that read token ids on the device share: the id storage,
// its checks, and multi-output bookkeeping.
#pragma once

#include <cuda_runtime.h>

#include <deque>
#include <initializer_list>

#include "tp_core.h"

namespace tp {

// Storage of token ids: every dtype is stored as float32, index outputs
// (argmax, the alternatives of tokenLogprobs) as int32.
enum { IDS_F32 = 0, IDS_I32 = 1 };

// f32 holds every whole number up to 2^24 exactly: tables and vocabularies
// beyond that could not be addressed by their own ids.
constexpr int64_t TOKEN_MAX_VOCAB = (int64_t)1 << 24;

// The id at position i; f32 ids are truncated toward zero, as toList decodes
// integer dtypes.  2^24 and above, NaN and the infinities come back as
// TOKEN_MAX_VOCAB, which is outside every vocabulary; -2^24 and below as -2^24.
__device__ __forceinline__ int token_id(const void* ids, int kind, int64_t i) {
  if (kind == IDS_I32) return static_cast<const int32_t*>(ids)[i];
  const float f = static_cast<const float*>(ids)[i];
  if (fabsf(f) < (float)TOKEN_MAX_VOCAB) return (int)f;
  return f < 0.0f && f > -INFINITY ? -(int)TOKEN_MAX_VOCAB : (int)TOKEN_MAX_VOCAB;
}

inline int ids_kind_of(const Tensor& t) { return t.phys == PHYS_I32 ? IDS_I32 : IDS_F32; }

inline void check_ids_kind(int kind, const char* what) {
  TP_REQUIRE(kind == IDS_F32 || kind == IDS_I32, "%s: ids_kind must be 0 (float32 values) or 1 (int32), got %d", what,
             kind);
}

inline void check_vocab(int64_t V, const char* what) {
  TP_REQUIRE(V >= 1 && V <= TOKEN_MAX_VOCAB, "%s: a vocabulary of %lld is outside [1, 2^24]", what, (long long)V);
}

// Every value of a caller's buffers is 4 bytes; nothing more is asked of them.
inline void check_aligned(std::initializer_list<const void*> buffers, const char* what) {
  for (const void* p : buffers) TP_REQUIRE(((uintptr_t)p & 3) == 0, "%s: a buffer is not 4-byte aligned", what);
}

// Output tensors of one call: freed again if the call throws before they are
// registered.
class Outputs {
 public:
  Tensor& add(const Tensor& t) {
    all_.push_back(t);
    return all_.back();
  }
  // registers each tensor in its handle; one the caller has no handle for is freed
  void emit_all(std::initializer_list<tp_handle*> to) {
    for (auto h = to.begin(); !all_.empty(); ++h) {
      if (*h) emit(all_.front(), *h);
      else dfree(all_.front().ptr);
      all_.pop_front();
    }
  }
  ~Outputs() {
    for (Tensor& t : all_)
      if (t.ptr) cudaFreeAsync(t.ptr, stream());
  }

 private:
  std::deque<Tensor> all_;
};

}  // namespace tp
