// dropout.cuh — dropout with a mask made from a counter, onto an optional residual.
//
//   y = keep(e) ? x * 1/(1 - p) : 0   (+ residual)
//
// in fp32, rounded once to the tensors' type.  keep(e) is dropout_mask.cuh's rule on
// the element's linear index, so the gradient (the same map applied to dy, without the
// residual) makes the mask again and nothing is stored.
//
// A pass moves 2 (3 with a residual) values per element and is bound by HBM.
#pragma once

#include <cuda_fp16.h>

#include "dropout_mask.cuh"
#include "sm100_common.cuh"

namespace fp8b {

struct DropoutParams {
  const void* x;
  const void* residual;  // nullptr: none
  void* y;
  const int64_t* seed;  // device scalar
  int64_t n;
  uint32_t thresh;  // p * 65536, rounded
  float scale;      // 1 / (1 - p); 0 for p = 1
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

constexpr int kDropoutThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kDropoutThreads) dropout_kernel(const DropoutParams p) {
  pdl_sync();
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  T* y = static_cast<T*>(p.y);
  const uint64_t seed = static_cast<uint64_t>(*p.seed);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x * 8;
  for (int64_t e0 = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 8; e0 < p.n; e0 += step) {
    const uint32_t keep = dropout_keep8(seed, e0, p.thresh);
    for (int k = 0; k < 8 && e0 + k < p.n; ++k) {
      float v = (keep >> k) & 1u ? to_f32(x[e0 + k]) * p.scale : 0.0f;
      if (res != nullptr) v += to_f32(res[e0 + k]);
      y[e0 + k] = from_f32<T>(v);
    }
  }
}

}  // namespace fp8b
