// embedding.cuh — token embedding with scaling, and its gradient by sorted tokens.
//
//   y_i = scale * W[id_i]                          (fp32, rounded once to y's type)
//   dW_v = scale * sum_{i : id_i = v} dy_i         (fp32, in token order; zero rows
//                                                   for tokens that do not occur and
//                                                   for the padding token)
//
// An id outside [0, vocab) reads nothing: its output row is zero, it adds to no
// gradient, and the device error word records kErrTokenRange.
#pragma once

#include "dropout.cuh"
#include "sm100_common.cuh"

namespace fp8b {

constexpr int kErrTokenRange = 201;  // a token id outside [0, vocab)

struct EmbedParams {
  const void* ids;
  int ids64;
  const void* weight;
  int64_t weight_stride;
  void* out;
  const void* dout;
  void* dweight;
  int64_t tokens, vocab, padding_idx;  // padding_idx < 0: none
  int width;
  float scale;
  int* err;
};

__device__ __forceinline__ int64_t load_id(const EmbedParams& p, int64_t i) {
  return p.ids64 ? static_cast<const int64_t*>(p.ids)[i] : static_cast<const int32_t*>(p.ids)[i];
}

template <typename TW, typename TO>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const EmbedParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; i < p.tokens;
       i += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
    const int64_t id = load_id(p, i);
    const bool valid = id >= 0 && id < p.vocab;
    if (!valid && lane == 0) record_error(p.err, kErrTokenRange);
    const TW* w = static_cast<const TW*>(p.weight) + (valid ? id : 0) * p.weight_stride;
    TO* o = static_cast<TO*>(p.out) + i * p.width;
    for (int c = lane; c < p.width; c += 32) o[c] = from_f32<TO>(valid ? to_f32(w[c]) * p.scale : 0.0f);
  }
}

// One warp per vocabulary row, which looks through all ids for its own.
template <typename TW, typename TO>
__global__ void __launch_bounds__(256) embed_bwd_simple_kernel(const EmbedParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  for (int64_t v = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; v < p.vocab;
       v += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
    TW* o = static_cast<TW*>(p.dweight) + v * p.width;
    for (int c0 = 0; c0 < p.width; c0 += 256) {
      float acc[8] = {};
      if (v != p.padding_idx)
        for (int64_t i0 = 0; i0 < p.tokens; i0 += 32) {
          unsigned hit = __ballot_sync(~0u, i0 + lane < p.tokens && load_id(p, i0 + lane) == v);
          while (hit) {
            const int64_t i = i0 + __ffs(hit) - 1;
            hit &= hit - 1;
            for (int k = 0; k < 8; ++k) {
              const int c = c0 + k * 32 + lane;
              if (c < p.width) acc[k] += to_f32(static_cast<const TO*>(p.dout)[i * p.width + c]);
            }
          }
        }
      for (int k = 0; k < 8; ++k) {
        const int c = c0 + k * 32 + lane;
        if (c < p.width) o[c] = from_f32<TW>(acc[k] * p.scale);
      }
    }
  }
}

}  // namespace fp8b
