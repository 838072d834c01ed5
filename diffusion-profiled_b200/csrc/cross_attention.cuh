// cross_attention.cuh — attention of a set of queries over an encoder's states.
//
//   s_ij = scale * q_i . k_j          over the kept keys j (key_lengths, key_mask)
//   p_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp(s_ij)
//   o_i  = sum_j p_ij v_j
// and its gradient
//   dv_j = sum_i p_ij do_i,  dp_ij = do_i . v_j,  delta_i = sum_j p_ij dp_ij,
//   ds_ij = p_ij (dp_ij - delta_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// with the sums over i running over the queries of every head that shares the keys.
// A query without kept keys has o = 0, lse = -inf and adds nothing to any gradient;
// what is stored at a key that is not kept (infinities and NaN too) is never used.
#pragma once

#include <cuda_fp16.h>

#include "dropout.cuh"
#include "sm100_common.cuh"

namespace fp8b {

struct XStrides {
  int64_t batch, token, head;  // elements
};

struct XAttnParams {
  const void *q, *k, *v, *o_in, *dout;
  void *o, *dq, *dk, *dv;
  XStrides sq, sk, sv, so, sdo, sdq, sdk, sdv;
  float* lse;    // [batch][heads][q_len]
  float* delta;  // same, backward
  const int32_t* key_lengths;
  const uint8_t* key_mask;
  int64_t mask_stride;
  int batch, q_len, k_len, heads, kv_heads, head_dim;
  float scale;
  int* err;
};

__device__ __forceinline__ int x_key_count(const XAttnParams& p, int b) {
  return p.key_lengths == nullptr ? p.k_len : max(0, min(p.k_len, p.key_lengths[b]));
}
__device__ __forceinline__ bool x_key_kept(const XAttnParams& p, int b, int j) {
  return p.key_mask == nullptr || p.key_mask[b * p.mask_stride + j] != 0;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// 4 consecutive head channels per lane (head_dim <= 128).
template <typename T>
__device__ __forceinline__ void x_load4(const T* row, int lane, int d, float (&f)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = lane * 4 + k < d ? to_f32(row[lane * 4 + k]) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void x_store4(T* row, int lane, int d, const float (&f)[4], float scale) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane * 4 + k < d) row[lane * 4 + k] = from_f32<T>(f[k] * scale);
}
__device__ __forceinline__ float dot4(const float (&a)[4], const float (&b)[4]) {
  return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
}

// One warp per query row.
template <typename T>
__global__ void __launch_bounds__(256) x_fwd_simple_kernel(const XAttnParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.heads * p.q_len;
  const int group = p.heads / p.kv_heads;
  for (int64_t r = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; r < rows;
       r += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
    const int i = static_cast<int>(r % p.q_len), h = static_cast<int>(r / p.q_len % p.heads),
              b = static_cast<int>(r / p.q_len / p.heads), hk = h / group;
    float q[4], o[4] = {}, m = -INFINITY, l = 0.0f;
    x_load4(static_cast<const T*>(p.q) + b * p.sq.batch + i * p.sq.token + h * p.sq.head, lane, p.head_dim, q);
    const int n = x_key_count(p, b);
    for (int j = 0; j < n; ++j) {
      if (!x_key_kept(p, b, j)) continue;
      float k[4], v[4];
      x_load4(static_cast<const T*>(p.k) + b * p.sk.batch + j * p.sk.token + hk * p.sk.head, lane, p.head_dim, k);
      x_load4(static_cast<const T*>(p.v) + b * p.sv.batch + j * p.sv.token + hk * p.sv.head, lane, p.head_dim, v);
      const float s = warp_sum(dot4(q, k)) * p.scale;
      const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.0f : expf(m - mn), w = expf(s - mn);
      l = l * f + w;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = o[c] * f + w * v[c];
      m = mn;
    }
    x_store4(static_cast<T*>(p.o) + b * p.so.batch + i * p.so.token + h * p.so.head, lane, p.head_dim, o,
             l > 0.0f ? 1.0f / l : 0.0f);
    if (p.lse != nullptr && lane == 0) p.lse[r] = l > 0.0f ? m + logf(l) : -INFINITY;
  }
}

// One warp per query row: delta and dq.
template <typename T>
__global__ void __launch_bounds__(256) x_dq_simple_kernel(const XAttnParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.heads * p.q_len;
  const int group = p.heads / p.kv_heads;
  for (int64_t r = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; r < rows;
       r += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
    const int i = static_cast<int>(r % p.q_len), h = static_cast<int>(r / p.q_len % p.heads),
              b = static_cast<int>(r / p.q_len / p.heads), hk = h / group;
    float q[4], g[4], o[4], dq[4] = {};
    x_load4(static_cast<const T*>(p.q) + b * p.sq.batch + i * p.sq.token + h * p.sq.head, lane, p.head_dim, q);
    x_load4(static_cast<const T*>(p.dout) + b * p.sdo.batch + i * p.sdo.token + h * p.sdo.head, lane, p.head_dim, g);
    x_load4(static_cast<const T*>(p.o_in) + b * p.so.batch + i * p.so.token + h * p.so.head, lane, p.head_dim, o);
    const float lse = p.lse[r], delta = warp_sum(dot4(g, o));
    const int n = lse == -INFINITY ? 0 : x_key_count(p, b);
    for (int j = 0; j < n; ++j) {
      if (!x_key_kept(p, b, j)) continue;
      float k[4], v[4];
      x_load4(static_cast<const T*>(p.k) + b * p.sk.batch + j * p.sk.token + hk * p.sk.head, lane, p.head_dim, k);
      x_load4(static_cast<const T*>(p.v) + b * p.sv.batch + j * p.sv.token + hk * p.sv.head, lane, p.head_dim, v);
      const float ds = expf(warp_sum(dot4(q, k)) * p.scale - lse) * (warp_sum(dot4(g, v)) - delta);
#pragma unroll
      for (int c = 0; c < 4; ++c) dq[c] += ds * k[c];
    }
    x_store4(static_cast<T*>(p.dq) + b * p.sdq.batch + i * p.sdq.token + h * p.sdq.head, lane, p.head_dim, dq, p.scale);
    if (lane == 0) p.delta[r] = delta;
  }
}

// One warp per key row: dk and dv over the queries of the heads that share it.
template <typename T>
__global__ void __launch_bounds__(256) x_dkv_simple_kernel(const XAttnParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.kv_heads * p.k_len;
  const int group = p.heads / p.kv_heads;
  for (int64_t r = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; r < rows;
       r += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
    const int j = static_cast<int>(r % p.k_len), hk = static_cast<int>(r / p.k_len % p.kv_heads),
              b = static_cast<int>(r / p.k_len / p.kv_heads);
    float dk[4] = {}, dv[4] = {};
    if (j < x_key_count(p, b) && x_key_kept(p, b, j)) {
      float k[4], v[4];
      x_load4(static_cast<const T*>(p.k) + b * p.sk.batch + j * p.sk.token + hk * p.sk.head, lane, p.head_dim, k);
      x_load4(static_cast<const T*>(p.v) + b * p.sv.batch + j * p.sv.token + hk * p.sv.head, lane, p.head_dim, v);
      for (int h = hk * group; h < (hk + 1) * group; ++h)
        for (int i = 0; i < p.q_len; ++i) {
          const int64_t row = (static_cast<int64_t>(b) * p.heads + h) * p.q_len + i;
          float q[4], g[4];
          x_load4(static_cast<const T*>(p.q) + b * p.sq.batch + i * p.sq.token + h * p.sq.head, lane, p.head_dim, q);
          x_load4(static_cast<const T*>(p.dout) + b * p.sdo.batch + i * p.sdo.token + h * p.sdo.head, lane, p.head_dim,
                  g);
          const float w = expf(warp_sum(dot4(q, k)) * p.scale - p.lse[row]);
          const float ds = w * (warp_sum(dot4(g, v)) - p.delta[row]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            dv[c] += w * g[c];
            dk[c] += ds * q[c];
          }
        }
    }
    x_store4(static_cast<T*>(p.dk) + b * p.sdk.batch + j * p.sdk.token + hk * p.sdk.head, lane, p.head_dim, dk, p.scale);
    x_store4(static_cast<T*>(p.dv) + b * p.sdv.batch + j * p.sdv.token + hk * p.sdv.head, lane, p.head_dim, dv, 1.0f);
  }
}

}  // namespace fp8b
