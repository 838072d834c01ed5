// dropout.cuh — dropout with a mask made from a counter, onto an optional residual.
//
//   y = keep(e) ? x * 1/(1 - p) : 0   (+ residual)
//
// in fp32, rounded once to the tensors' type.  keep(e) is dropout_mask.cuh's rule on
// the element's linear index, so the gradient (the same map applied to dy, without the
// residual) makes the mask again and nothing is stored.
//
// A pass moves 2 (3 with a residual) values per element and is bound by HBM; the mask
// takes about six integer operations an element.  A thread takes 8 elements (one or two
// 16-byte loads a tensor, two generator words) twice a round, its second 8 a grid's width
// on, so that enough loads are in flight.  16,385 x 4093 fp32: 95.6 us a pass, 5.6 TB/s,
// 86 % of the measured copy rate; 131,072 x 128 bf16 onto a residual: 18.8 us, 5.4 TB/s.
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

// 8 consecutive values as 16-byte words (16-byte aligned).
template <typename T>
struct Words8 {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Words8<T> load_words8(const T* p) {
  Words8<T> v;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) v.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return v;
}
// The same of memory that the kernel may write too (not by the read-only path).
template <typename T>
__device__ __forceinline__ Words8<T> load_own_words8(const T* p) {
  Words8<T> v;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) v.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return v;
}
template <typename T>
__device__ __forceinline__ void widen8(const Words8<T>& v, float (&f)[8]) {
  const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = to_f32(t[k]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  Words8<T> v;
  T* t = reinterpret_cast<T*>(&v);
#pragma unroll
  for (int k = 0; k < 8; ++k) t[k] = from_f32<T>(f[k]);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = v.w[i];
}

constexpr int kDropoutThreads = 256;

// VEC: the pointers are 16-byte aligned.  y may be x or the residual: each value is read by the thread that writes it.
template <typename T, bool VEC, bool RESIDUAL>
__global__ void __launch_bounds__(kDropoutThreads) dropout_kernel(const DropoutParams p) {
  pdl_sync();
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  T* y = static_cast<T*>(p.y);
  const uint64_t seed = static_cast<uint64_t>(*p.seed);
  const int64_t threads = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t whole = VEC ? p.n / 8 : 0;  // groups of 8 elements
  constexpr int kAtOnce = 2;
  for (int64_t g0 = me; g0 < whole; g0 += kAtOnce * threads) {
    Words8<T> xv[kAtOnce], rv[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int64_t g = g0 + u * threads;
      if (g >= whole) continue;
      xv[u] = load_own_words8(x + g * 8);
      if (RESIDUAL) rv[u] = load_own_words8(res + g * 8);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int64_t g = g0 + u * threads;
      if (g >= whole) continue;
      const uint32_t keep = dropout_keep8(seed, g * 8, p.thresh);
      float f[8], r[8];
      widen8(xv[u], f);
      if (RESIDUAL) widen8(rv[u], r);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f[k] = (keep >> k) & 1u ? f[k] * p.scale : 0.0f;
        if (RESIDUAL) f[k] += r[k];
      }
      store8(y + g * 8, f);
    }
  }
  // the rest, element by element (everything where a pointer is not aligned)
  for (int64_t g = whole + me; g * 8 < p.n; g += threads) {
    const uint32_t keep = dropout_keep8(seed, g * 8, p.thresh);
    for (int k = 0; k < 8 && g * 8 + k < p.n; ++k) {
      const int64_t e = g * 8 + k;
      float v = (keep >> k) & 1u ? to_f32(x[e]) * p.scale : 0.0f;
      if (RESIDUAL) v += to_f32(res[e]);
      y[e] = from_f32<T>(v);
    }
  }
}

}  // namespace fp8b
