// embedding.cuh — token embedding with scaling, and its gradient by sorted tokens.
//
//   y_i = scale * W[id_i]                          (fp32, rounded once to y's type)
//   dW_v = scale * sum_{i : id_i = v} dy_i         (fp32; zero rows for tokens that do
//                                                   not occur and for the padding token)
//
// An id outside [0, vocab) reads nothing: its output row is zero, it adds to no
// gradient, and the device error word records kErrTokenRange.
//
// Gradient, three launches:
//   1. embed_sort_kernel sorts (id, position) by id, stably, in radix passes of up to 9
//      bits inside one cooperative launch (a token's key is its id; padding and ids out of
//      range take the key `vocab`, behind all others), and finds each row's first place;
//   2. embed_sum_kernel sums the gradient rows in that order.  The sorted tokens are cut
//      into chunks of equal length whatever the ids, so that a token that is half of the
//      batch is summed by many warps; a row whose tokens lie in one chunk is written at
//      once, the others leave one partial sum (fp32) a chunk.  Rows without tokens are
//      zeroed by the same launch;
//   3. embed_join_kernel adds the partial sums of each row that crosses chunks, in order.
// The order of every sum follows from the ids alone: no float atomics, the same bits
// every time.  The launches are bound by the bytes of dy and dW; the sort moves 16 bytes a
// token and pass.
#pragma once

#include "dropout.cuh"
#include "sm100_common.cuh"

namespace fp8b {

constexpr int kErrTokenRange = 201;   // a token id outside [0, vocab)
constexpr int kErrTimeoutSort = 202;  // a CTA gave up waiting for the others between two passes

struct EmbedParams {
  const void* ids;
  int ids64;
  const void* weight;
  int64_t weight_stride;
  void* out;
  int64_t tokens, vocab;
  int width;
  float scale;
  int* err;
};

__device__ __forceinline__ int64_t load_id(const void* ids, int ids64, int64_t i) {
  return ids64 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// ============================================================================ lookup
// One warp per token; VEC: rows of whole 16-byte words (width % 8 == 0, aligned).
template <typename TW, typename TO, bool VEC>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const EmbedParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; i < p.tokens; i += warps) {
    const int64_t id = load_id(p.ids, p.ids64, i);
    const bool valid = id >= 0 && id < p.vocab;
    if (!valid && lane == 0) record_error(p.err, kErrTokenRange);
    const TW* w = static_cast<const TW*>(p.weight) + (valid ? id : 0) * p.weight_stride;
    TO* o = static_cast<TO*>(p.out) + i * p.width;
    if constexpr (VEC) {
      constexpr int kAtOnce = 4;  // 1024 channels' loads in flight
      for (int c0 = lane * 8; c0 < p.width; c0 += 256 * kAtOnce) {
        Words8<TW> v[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
          if (c0 + 256 * u < p.width) v[u] = load_words8(w + c0 + 256 * u);
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
          if (c0 + 256 * u < p.width) {
            float f[8];
            widen8(v[u], f);
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = valid ? f[k] * p.scale : 0.0f;
            store8(o + c0 + 256 * u, f);
          }
      }
    } else {
      for (int c = lane; c < p.width; c += 32) o[c] = from_f32<TO>(valid ? to_f32(w[c]) * p.scale : 0.0f);
    }
  }
}

// ============================================================================ sort
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxBits = 9;  // 512 digits: one count a warp and digit fits shared memory (64 KB)
constexpr int kSortMaxCtas = 64;

struct EmbedSortParams {
  const void* ids;
  int ids64;
  int64_t vocab, padding_idx;
  int tokens;
  int passes, bits;        // digits of `bits` bits, least significant first
  int per_cta, per_warp;   // tokens, multiples of 32
  uint32_t* key[2];
  uint32_t* pos[2];
  uint32_t* counts;        // [gridDim.x][1 << bits]
  uint32_t* row_start;     // [vocab + 1]: first place whose key is at least the row
  unsigned int *arrive, *depart;  // zero between launches
  int* err;
};

// All CTAs' writes so far are visible to all.  `round` counts the barriers of the launch from 1.
__device__ __forceinline__ bool sort_barrier(const EmbedSortParams& p, unsigned int round) {
  __shared__ int passed;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    red_release_gpu_add_u32(p.arrive, 1u);
    const uint64_t t0 = globaltimer_ns();
    int ok = 1;
    while (ld_acquire_gpu_u32(p.arrive) < round * gridDim.x) {
      if (globaltimer_ns() - t0 > FP8_WAIT_TIMEOUT_NS) {
        record_error(p.err, kErrTimeoutSort);
        ok = 0;
        break;
      }
    }
    __threadfence();
    passed = ok;
  }
  __syncthreads();
  return passed != 0;
}

__global__ void __launch_bounds__(kSortThreads, 1) embed_sort_kernel(const EmbedSortParams p) {
  extern __shared__ uint32_t sort_smem[];
  uint32_t* warp_count = sort_smem;                                // [kSortWarps][digits]
  uint32_t* base = sort_smem + kSortWarps * (1 << p.bits);         // [digits]
  uint32_t* scan = base + (1 << p.bits);                           // [kSortWarps]
  pdl_sync();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int digits = 1 << p.bits;
  const int begin = min(p.tokens, static_cast<int>(blockIdx.x) * p.per_cta + warp * p.per_warp);
  const int end = min(min(p.tokens, (static_cast<int>(blockIdx.x) + 1) * p.per_cta), begin + p.per_warp);
  uint32_t* mine = warp_count + warp * digits;
  unsigned int round = 0;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const uint32_t* key_in = p.key[(pass + 1) & 1];
    const uint32_t* pos_in = p.pos[(pass + 1) & 1];
    uint32_t* key_out = p.key[pass & 1];
    uint32_t* pos_out = p.pos[pass & 1];
    const auto key_of = [&](int i) -> uint32_t {
      if (pass > 0) return __ldcg(key_in + i);
      const int64_t id = load_id(p.ids, p.ids64, i);
      return id < 0 || id >= p.vocab || id == p.padding_idx ? static_cast<uint32_t>(p.vocab) : static_cast<uint32_t>(id);
    };
    // ---- this warp's count of each digit over its own stretch of tokens
    for (int d = lane; d < digits; d += 32) mine[d] = 0;
    __syncwarp();
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const bool in = i < end;
      const uint32_t d = in ? (key_of(i) >> shift) & (digits - 1) : ~0u;
      const unsigned same = __match_any_sync(~0u, d);
      if (in && (same & ((1u << lane) - 1)) == 0) mine[d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    // ---- the CTA's count, and each warp's place among the CTA's tokens of the digit
    if (tid < digits) {
      uint32_t sum = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = warp_count[w * digits + tid];
        warp_count[w * digits + tid] = sum;
        sum += c;
      }
      p.counts[blockIdx.x * digits + tid] = sum;
    }
    if (!sort_barrier(p, ++round)) return;
    // ---- where the digit begins, and the tokens of the CTAs before this one in it
    uint32_t before = 0, total = 0;
    if (tid < digits)
#pragma unroll 8
      for (int c = 0; c < static_cast<int>(gridDim.x); ++c) {
        const uint32_t n = __ldcg(p.counts + c * digits + tid);
        before += c < static_cast<int>(blockIdx.x) ? n : 0u;
        total += n;
      }
    uint32_t incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      uint32_t v = scan[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += u;
      }
      scan[lane] = v;
    }
    __syncthreads();
    if (tid < digits) base[tid] = (warp > 0 ? scan[warp - 1] : 0u) + incl - total + before;
    __syncthreads();
    // ---- to their places, in order
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const bool in = i < end;
      const uint32_t key = in ? key_of(i) : 0u;
      const uint32_t d = in ? (key >> shift) & (digits - 1) : ~0u;
      const unsigned same = __match_any_sync(~0u, d);
      const int rank = __popc(same & ((1u << lane) - 1));
      if (in) {
        const uint32_t to = base[d] + mine[d] + rank;
        key_out[to] = key;
        pos_out[to] = pass > 0 ? __ldcg(pos_in + i) : static_cast<uint32_t>(i);
      }
      __syncwarp();
      if (in && rank == 0) mine[d] += __popc(same);
      __syncwarp();
    }
    if (!sort_barrier(p, ++round)) return;
  }
  // ---- each row's first place, by bisection
  const uint32_t* key = p.key[(p.passes + 1) & 1];
  for (int64_t v = static_cast<int64_t>(blockIdx.x) * kSortThreads + tid; v <= p.vocab;
       v += static_cast<int64_t>(gridDim.x) * kSortThreads) {
    int lo = 0, hi = p.tokens;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldcg(key + mid) < static_cast<uint32_t>(v)) lo = mid + 1;
      else hi = mid;
    }
    p.row_start[v] = static_cast<uint32_t>(lo);
  }
  // the last CTA to leave sets the counters back
  __syncthreads();
  if (tid == 0 && atom_add_acq_rel_gpu_u32(p.depart, 1u) == gridDim.x - 1) {
    *p.arrive = 0u;
    *p.depart = 0u;
  }
}

// ============================================================================ sums
constexpr int kSumSlice = 256;  // channels of a warp's work: 8 a lane

struct EmbedSumParams {
  const uint32_t *key, *pos, *row_start;  // sorted; rows' first places [vocab + 1]
  const void* dout;
  void* dweight;
  float *head, *tail;  // [chunks][width]: sums of the row that began before the chunk / that goes on after it
  int64_t vocab;
  int chunk;   // sorted tokens of a chunk
  int slices;  // warps' shares of a row: ceil(width / 256)
  int width;
  float scale;
};

// This lane's 8 channels of a slice: consecutive (VEC) or every 32nd.
template <bool VEC>
__device__ __forceinline__ int slice_channel(int slice, int lane, int k) {
  return slice * kSumSlice + (VEC ? lane * 8 + k : k * 32 + lane);
}
template <typename T, bool VEC>
__device__ __forceinline__ void slice_load(const T* row, int slice, int lane, int width, float (&f)[8]) {
  if constexpr (VEC) {
    const int c = slice_channel<true>(slice, lane, 0);
    if (c < width) {
      widen8(load_words8(row + c), f);
      return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 0.0f;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = slice_channel<false>(slice, lane, k);
      f[k] = c < width ? to_f32(row[c]) : 0.0f;
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void slice_store(T* row, int slice, int lane, int width, const float (&f)[8]) {
  if constexpr (VEC) {
    const int c = slice_channel<true>(slice, lane, 0);
    if (c < width) store8(row + c, f);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = slice_channel<false>(slice, lane, k);
      if (c < width) row[c] = from_f32<T>(f[k]);
    }
  }
}

template <typename TW, typename TO, bool VEC>
__global__ void __launch_bounds__(256) embed_sum_kernel(const EmbedSumParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  const int64_t me = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int live = static_cast<int>(p.row_start[p.vocab]);  // padding and ids out of range lie behind
  const int64_t sums = static_cast<int64_t>((live + p.chunk - 1) / p.chunk) * p.slices;
  const TO* dout = static_cast<const TO*>(p.dout);
  TW* dw = static_cast<TW*>(p.dweight);
  for (int64_t item = me; item < sums; item += warps) {
    const int chunk = static_cast<int>(item / p.slices), slice = static_cast<int>(item % p.slices);
    const int begin = chunk * p.chunk, end = min(live, begin + p.chunk);
    float acc[8] = {};
    uint32_t row = p.key[begin];
    bool first = begin > 0 && p.key[begin - 1] == row;  // the row began in an earlier chunk
    const auto flush = [&](bool goes_on) {
      if (first || goes_on) {
        float* part = (first ? p.head : p.tail) + static_cast<int64_t>(chunk) * p.width;
        slice_store<float, VEC>(part, slice, lane, p.width, acc);
      } else {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = acc[k] * p.scale;
        slice_store<TW, VEC>(dw + static_cast<int64_t>(row) * p.width, slice, lane, p.width, f);
      }
    };
    for (int p0 = begin; p0 < end; p0 += 32) {
      const int n = min(32, end - p0);
      const uint32_t my_key = lane < n ? p.key[p0 + lane] : 0u, my_pos = lane < n ? p.pos[p0 + lane] : 0u;
      constexpr int kAtOnce = 4;  // rows in flight
      for (int u0 = 0; u0 < n; u0 += kAtOnce) {
        float f[kAtOnce][8];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const uint32_t pos = __shfl_sync(~0u, my_pos, (u0 + u) & 31);
          if (u0 + u < n) slice_load<TO, VEC>(dout + static_cast<int64_t>(pos) * p.width, slice, lane, p.width, f[u]);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const uint32_t key = __shfl_sync(~0u, my_key, (u0 + u) & 31);
          if (u0 + u >= n) continue;
          if (key != row) {
            flush(false);
            row = key;
            first = false;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] += f[u][k];
        }
      }
    }
    flush(end < live && p.key[end] == row);
  }
  // rows without tokens
  for (int64_t v = me; v < p.vocab; v += warps) {
    if (p.row_start[v] != p.row_start[v + 1]) continue;
    const float zero[8] = {};
    for (int slice = 0; slice < p.slices; ++slice) slice_store<TW, VEC>(dw + v * p.width, slice, lane, p.width, zero);
  }
}

// Rows that cross chunks: the partial sum of the chunk the row begins in, then those of the chunks it goes on in.
template <typename TW, bool VEC>
__global__ void __launch_bounds__(256) embed_join_kernel(const EmbedSumParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  const int live = static_cast<int>(p.row_start[p.vocab]);
  const int64_t items = static_cast<int64_t>((live + p.chunk - 1) / p.chunk) * p.slices;
  for (int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; item < items; item += warps) {
    const int chunk = static_cast<int>(item / p.slices), slice = static_cast<int>(item % p.slices);
    const int end = (chunk + 1) * p.chunk;
    if (end >= live) continue;
    const uint32_t row = p.key[end];
    if (p.key[end - 1] != row || static_cast<int>(p.row_start[row]) < chunk * p.chunk) continue;  // ends here, or began before
    const int last = (static_cast<int>(p.row_start[row + 1]) - 1) / p.chunk;
    float acc[8];
    slice_load<float, VEC>(p.tail + static_cast<int64_t>(chunk) * p.width, slice, lane, p.width, acc);
    constexpr int kAtOnce = 4;
    for (int c0 = chunk + 1; c0 <= last; c0 += kAtOnce) {
      float f[kAtOnce][8];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (c0 + u <= last) slice_load<float, VEC>(p.head + static_cast<int64_t>(c0 + u) * p.width, slice, lane, p.width, f[u]);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (c0 + u <= last)
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] += f[u][k];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] *= p.scale;
    slice_store<TW, VEC>(static_cast<TW*>(p.dweight) + static_cast<int64_t>(row) * p.width, slice, lane, p.width, acc);
  }
}

}  // namespace fp8b
