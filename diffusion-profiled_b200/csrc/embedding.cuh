// embedding.cuh — token embedding with scaling, and its gradient by sorted tokens.
//
//   y_i = scale * W[id_i]                          (fp32, rounded once to y's type)
//   dW_v = scale * sum_{i : id_i = v} dy_i         (fp32; zero rows for tokens that do
//                                                   not occur and for the padding token)
//
// An id outside [0, vocab) reads nothing: its output row is zero, the lookup records
// kErrTokenRange in the device error word, and it adds to no gradient.
//
// Gradient of few tokens, one launch (embed_few_kernel): every token looks through all ids
// for its row's others, and the first of a row sums them.  Of more tokens, three launches:
//   1. embed_sort_kernel sorts (id, position) by id, stably, in radix passes of up to 9
//      bits inside one cooperative launch (a token's key is its id; padding and ids out of
//      range take the key `vocab`, behind all others), and marks the rows that occur;
//   2. embed_sum_kernel sums the gradient rows in that order.  The sorted tokens are cut
//      into chunks of equal length whatever the ids, so that a token that is half of the
//      batch is summed by many warps; a row whose tokens lie in one chunk is written at
//      once, the others leave one partial sum (fp32) a chunk.  Rows without tokens are
//      zeroed by the same launch;
//   3. embed_join_kernel adds the partial sums of each row that crosses chunks, in order.
// The order of every sum follows from the ids alone: no float atomics, the same bits
// every time.  The launches are bound by the bytes of dy and dW; the sort moves 16 bytes a
// token and pass.  262,147 tokens of 1024 channels (bf16) over 131,072 rows: lookup 117 us,
// sort 36, sums 158 (805 MB, 5.1 TB/s), join 20: 332 us against 246 of bytes.
#pragma once

#include <type_traits>

#include "dropout.cuh"
#include "sm100_common.cuh"

namespace fp8b {

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
// A warp takes two tokens a step, so that two rows' loads are in flight; VEC: rows of whole 16-byte words (width % 8
// == 0, aligned).
template <typename TW, typename TO, bool VEC>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const EmbedParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  constexpr int kTokens = 2;
  for (int64_t i0 = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; i0 < p.tokens;
       i0 += kTokens * warps) {
    const TW* w[kTokens];
    TO* o[kTokens];
    bool there[kTokens], valid[kTokens];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      const int64_t i = i0 + t * warps;
      there[t] = i < p.tokens;
      const int64_t id = there[t] ? load_id(p.ids, p.ids64, i) : 0;
      valid[t] = id >= 0 && id < p.vocab;
      if (!valid[t] && lane == 0) record_error(p.err, kErrTokenRange);
      w[t] = static_cast<const TW*>(p.weight) + (valid[t] ? id : 0) * p.weight_stride;
      o[t] = static_cast<TO*>(p.out) + (there[t] ? i : 0) * p.width;
    }
    if constexpr (VEC) {
      constexpr int kAtOnce = 2;  // 512 channels of each token
      for (int c0 = lane * 8; c0 < p.width; c0 += 256 * kAtOnce) {
        Words8<TW> v[kTokens][kAtOnce];
#pragma unroll
        for (int t = 0; t < kTokens; ++t)
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u)
            if (there[t] && c0 + 256 * u < p.width) v[t][u] = load_words8(w[t] + c0 + 256 * u);
#pragma unroll
        for (int t = 0; t < kTokens; ++t)
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u)
            if (there[t] && c0 + 256 * u < p.width) {
              float f[8];
              widen8(v[t][u], f);
#pragma unroll
              for (int k = 0; k < 8; ++k) f[k] = valid[t] ? f[k] * p.scale : 0.0f;
              store8(o[t] + c0 + 256 * u, f);
            }
      }
    } else {
      // 16-bit outputs in pairs from the row's first 4-byte boundary on, so that a warp's store fills whole sectors but
      // for its ends (100,000 x 777 bf16: 67 us, with 2-byte stores 108)
      constexpr int kPer = sizeof(TO) == 2 ? 2 : 1, kAtOnce = 8 / kPer;  // 256 channels of each token
      int head[kTokens];
#pragma unroll
      for (int t = 0; t < kTokens; ++t) head[t] = kPer == 2 ? (reinterpret_cast<uintptr_t>(o[t]) >> 1) & 1 : 0;
      for (int c0 = lane * kPer; c0 < p.width; c0 += 256) {
        TW v[kTokens][kAtOnce][kPer];
#pragma unroll
        for (int t = 0; t < kTokens; ++t)
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
              const int c = head[t] + c0 + 32 * kPer * u;
              if (there[t] && c + kPer <= p.width) v[t][u][k] = w[t][c + k];
            }
#pragma unroll
        for (int t = 0; t < kTokens; ++t)
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int c = head[t] + c0 + 32 * kPer * u;
            if (!there[t] || c + kPer > p.width) continue;
            struct alignas(sizeof(TO) * kPer) {
              TO x[kPer];
            } out;
#pragma unroll
            for (int k = 0; k < kPer; ++k) out.x[k] = from_f32<TO>(valid[t] ? to_f32(v[t][u][k]) * p.scale : 0.0f);
            *reinterpret_cast<decltype(out)*>(o[t] + c) = out;
          }
      }
      if constexpr (kPer == 2)  // the row's first and last value where they are not of a pair
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
          const int c = lane == 0 ? 0 : p.width - 1;
          if (there[t] && ((lane == 0 && head[t] == 1) || (lane == 1 && p.width > head[t] && ((p.width - head[t]) & 1))))
            o[t][c] = from_f32<TO>(valid[t] ? to_f32(w[t][c]) * p.scale : 0.0f);
        }
    }
  }
}

// ============================================================================ sort
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxBits = 9;  // 512 digits: one count a warp and digit fits shared memory (64 KB)
constexpr int kSortMaxCtas = 96;
constexpr int kSortAhead = 8;    // steps of 32 tokens whose keys are loaded together

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
  uint32_t* live;          // number of keys below vocab; zero when the launch starts, and so it stays if a CTA gives up
  uint32_t* present;       // bit v: row v occurs; [vocab / 32 + 1] words
  unsigned int* arrive;    // the call's own, zero when the launch starts
  unsigned int meet;       // CTAs that a barrier waits for: gridDim.x (more in the self-test, for a wait that runs out)
  uint64_t limit_ns;       // and how long it waits
  int* err;
};

// The lanes whose digit (of `bits` bits) is this lane's, among the lanes with `in` (one vote a bit: a quarter of the
// time of a match instruction over 32 different digits).
__device__ __forceinline__ unsigned same_digit(uint32_t d, int bits, bool in) {
  unsigned same = __ballot_sync(~0u, in);
#pragma unroll
  for (int b = 0; b < kSortMaxBits; ++b)
    if (b < bits) {
      const bool one = (d >> b) & 1u;
      const unsigned ones = __ballot_sync(~0u, one);
      same &= one ? ones : ~ones;
    }
  return same;
}

// All CTAs' writes so far are visible to all.  `round` counts the barriers of the launch from 1.  A CTA that gives up
// leaves: none of the others passes a later barrier, so `live` stays zero unless the keys are sorted, and the launches
// behind sum nothing (they never read keys that were not written).
__device__ __forceinline__ bool sort_barrier(const EmbedSortParams& p, unsigned int round) {
  __shared__ int passed;
  __syncthreads();
  if (p.meet == 1) return true;
  if (threadIdx.x == 0) {
    red_release_gpu_add_u32(p.arrive, 1u);  // with what the CTA's other threads wrote before the barrier above
    const uint64_t t0 = globaltimer_ns();
    int ok = 1;
    while (ld_acquire_gpu_u32(p.arrive) < round * p.meet) {
      if (globaltimer_ns() - t0 > p.limit_ns) {
        record_error(p.err, kErrTimeoutSort);
        ok = 0;
        break;
      }
    }
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
  const int64_t all = static_cast<int64_t>(gridDim.x) * kSortThreads, me = static_cast<int64_t>(blockIdx.x) * kSortThreads + tid;
  for (int64_t w = me; w <= p.vocab / 32; w += all) p.present[w] = 0;  // set after the passes' barriers
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
    for (int i0 = begin; i0 < end; i0 += 32 * kSortAhead) {
      uint32_t key[kSortAhead];
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) key[u] = i0 + 32 * u + lane < end ? key_of(i0 + 32 * u + lane) : 0u;
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        if (i0 + 32 * u >= end) break;
        const bool in = i0 + 32 * u + lane < end;
        const uint32_t d = (key[u] >> shift) & (digits - 1);
        const unsigned same = same_digit(d, p.bits, in);
        if (in && (same & ((1u << lane) - 1)) == 0) mine[d] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    // ---- the CTA's count, and each warp's place among the CTA's tokens of the digit
    if (tid < digits) {
      uint32_t c[kSortWarps], sum = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) c[w] = warp_count[w * digits + tid];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        warp_count[w * digits + tid] = sum;
        sum += c[w];
      }
      p.counts[blockIdx.x * digits + tid] = sum;
    }
    if (!sort_barrier(p, ++round)) return;
    // ---- where the digit begins, and the tokens of the CTAs before this one in it
    uint32_t before = 0, total = 0;
    if (tid < digits)
#pragma unroll 16
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
    for (int i0 = begin; i0 < end; i0 += 32 * kSortAhead) {
      uint32_t key[kSortAhead], pos[kSortAhead];
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        const int i = i0 + 32 * u + lane;
        key[u] = i < end ? key_of(i) : 0u;
        pos[u] = pass > 0 && i < end ? __ldcg(pos_in + i) : static_cast<uint32_t>(i);
      }
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        if (i0 + 32 * u >= end) break;
        const bool in = i0 + 32 * u + lane < end;
        const uint32_t d = (key[u] >> shift) & (digits - 1);
        const unsigned same = same_digit(d, p.bits, in);
        const int rank = __popc(same & ((1u << lane) - 1));
        if (in) {
          const uint32_t to = base[d] + mine[d] + rank;
          key_out[to] = key[u];
          pos_out[to] = pos[u];
        }
        __syncwarp();
        if (in && rank == 0) mine[d] += __popc(same);
        __syncwarp();
      }
    }
    if (!sort_barrier(p, ++round)) return;
  }
  // ---- the rows that occur: each where its key first does
  const uint32_t* key = p.key[(p.passes + 1) & 1];
  for (int64_t i0 = me; i0 <= p.tokens; i0 += 4 * all) {
    uint32_t k[4], before[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = i0 + u * all;
      k[u] = i < p.tokens ? __ldcg(key + i) : static_cast<uint32_t>(p.vocab);
      before[u] = i > 0 && i <= p.tokens ? __ldcg(key + i - 1) : ~0u;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = i0 + u * all;
      if (i > p.tokens || (i > 0 && k[u] == before[u])) continue;
      if (k[u] < p.vocab) atomicOr(p.present + (k[u] >> 5), 1u << (k[u] & 31));
      else if (i == 0 || before[u] < p.vocab) *p.live = static_cast<uint32_t>(i);
    }
  }
}

// ============================================================================ sums
constexpr int kSumSlice = 256;  // channels of a warp's work: 8 a lane

struct EmbedSumParams {
  const uint32_t *key, *pos;  // sorted
  const uint32_t *live, *present;
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
// The 8 channels as loaded (widened only when they are added: loads in flight take half the registers).  16-bit values
// that are loaded one by one stay in a register each: to pack two, the warp would wait for them (100,000 x 777 bf16:
// 66 us, packed 147).
template <typename T, bool VEC>
struct SliceWords {
  Words8<T> w;
};
template <typename T>
struct SliceWords<T, false> {
  uint32_t r[8];
};
template <typename T, bool VEC>
__device__ __forceinline__ SliceWords<T, VEC> slice_load(const T* row, int slice, int lane, int width) {
  SliceWords<T, VEC> v;
  if constexpr (VEC) {
    const int c = slice_channel<true>(slice, lane, 0);
    if (c < width) {
      v.w = load_words8(row + c);
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) v.w.w[i] = make_uint4(0, 0, 0, 0);
    }
  } else {
    using Bits = std::conditional_t<sizeof(T) == 2, unsigned short, uint32_t>;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = slice_channel<false>(slice, lane, k);
      v.r[k] = c < width ? __ldg(reinterpret_cast<const Bits*>(row) + c) : 0u;
    }
  }
  return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ void slice_widen(const SliceWords<T, VEC>& v, float (&f)[8]) {
  if constexpr (VEC) {
    widen8(v.w, f);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (sizeof(T) == 4) f[k] = __uint_as_float(v.r[k]);
      else if constexpr (std::is_same_v<T, __half>) f[k] = __half2float(__ushort_as_half(static_cast<unsigned short>(v.r[k])));
      else f[k] = __uint_as_float(v.r[k] << 16);
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
  const int live = static_cast<int>(*p.live);  // padding and ids out of range lie behind
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
    // Batches of kAtOnce rows; the next batch's loads are under way while this one is added.
    constexpr int kAtOnce = 4;
    SliceWords<TO, VEC> rows[2][kAtOnce];
    uint32_t my_key = 0, my_pos = 0;
    const auto fetch = [&](int at, SliceWords<TO, VEC>(&to)[kAtOnce]) {
      if (((at - begin) & 31) == 0 && at < end) my_pos = at + lane < end ? p.pos[at + lane] : 0u;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const uint32_t pos = __shfl_sync(~0u, my_pos, (at - begin + u) & 31);
        if (at + u < end) to[u] = slice_load<TO, VEC>(dout + static_cast<int64_t>(pos) * p.width, slice, lane, p.width);
      }
    };
    fetch(begin, rows[0]);
    for (int at0 = begin; at0 < end; at0 += 2 * kAtOnce)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int at = at0 + half * kAtOnce;
        if (at >= end) break;
        if (((at - begin) & 31) == 0) my_key = at + lane < end ? p.key[at + lane] : 0u;
        fetch(at + kAtOnce, rows[1 - half]);
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const uint32_t key = __shfl_sync(~0u, my_key, (at - begin + u) & 31);
          if (at + u >= end) continue;
          if (key != row) {
            flush(false);
            row = key;
            first = false;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
          }
          float f[8];
          slice_widen<TO, VEC>(rows[half][u], f);
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] += f[k];
        }
      }
    flush(end < live && p.key[end] == row);
  }
  // rows without tokens, 8 rows a warp and step
  for (int64_t v0 = me * 8; v0 < p.vocab; v0 += warps * 8) {
    uint32_t absent = ~(p.present[v0 >> 5] >> (v0 & 31)) & 0xffu;
    if (p.vocab - v0 < 8) absent &= (1u << (p.vocab - v0)) - 1;
    const float zero[8] = {};
    while (absent) {
      const int64_t v = v0 + __ffs(absent) - 1;
      absent &= absent - 1;
      for (int slice = 0; slice < p.slices; ++slice) slice_store<TW, VEC>(dw + v * p.width, slice, lane, p.width, zero);
    }
  }
}

// Rows that cross chunks: the partial sum of the chunk the row begins in, then those of the chunks it goes on in.  A
// warp takes 128 channels (4 a lane), 8 partial sums in flight: a row that is a twentieth of a long batch has over a
// hundred, but most warps find that their chunk begins none.  (262,147 tokens: 4 in flight 28 us, 8 20, 16 23, 32 28.)
constexpr int kJoinSlice = 128;
template <typename TW>
__global__ void __launch_bounds__(256) embed_join_kernel(const EmbedSumParams p) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  const int live = static_cast<int>(*p.live);
  const int slices = (p.width + kJoinSlice - 1) / kJoinSlice;
  const int64_t items = static_cast<int64_t>((live + p.chunk - 1) / p.chunk) * slices;
  for (int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; item < items; item += warps) {
    const int chunk = static_cast<int>(item / slices), c0 = static_cast<int>(item % slices) * kJoinSlice + lane;
    const int begin = chunk * p.chunk, end = begin + p.chunk;
    if (end >= live) continue;
    const uint32_t row = p.key[end];
    if (p.key[end - 1] != row || (begin > 0 && p.key[begin - 1] == row)) continue;  // ends here, or began before
    int last = chunk;  // the last chunk that begins with the row: 32 are looked at at a time
    for (unsigned more = ~0u; more == ~0u; last += __popc(more)) {
      const int64_t at = (static_cast<int64_t>(last) + 1 + lane) * p.chunk;
      more = __ballot_sync(~0u, at < live && p.key[at] == row);
    }
    const auto part = [&](const float* from, int of, float(&f)[4]) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        f[k] = c0 + 32 * k < p.width ? from[static_cast<int64_t>(of) * p.width + c0 + 32 * k] : 0.0f;
    };
    float acc[4];
    part(p.tail, chunk, acc);
    constexpr int kAtOnce = 8;
    for (int of = chunk + 1; of <= last; of += kAtOnce) {
      float f[kAtOnce][4];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (of + u <= last) part(p.head, of + u, f[u]);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (of + u <= last)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[k] += f[u][k];
    }
    TW* to = static_cast<TW*>(p.dweight) + static_cast<int64_t>(row) * p.width;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c0 + 32 * k < p.width) to[c0 + 32 * k] = from_f32<TW>(acc[k] * p.scale);
  }
}

// ============================================================================ few tokens
// Every token reads all ids: tokens^2 comparisons, but no sort, no workspace and two launches less.  Gradient of 77
// tokens of 64 channels, 32,768 rows: 4 us (16 us sorted); of 1024: 6 us (21), or 23 (25) where all are the same
// token, which one CTA a slice then sums; of 2048 the same token: 43 (35).  Rows of no whole 16-byte words cost the
// most: 777 channels, 1024 tokens 29 (40), the same token 74 (45).
constexpr int kFewTokens = 1024;
constexpr int kFewThreads = 256;
constexpr int kFewRows = 64;  // rows that a CTA looks for at a time, to zero those without tokens

struct EmbedFewParams {
  const void* ids;
  int ids64;
  int tokens;
  const void* dout;
  void* dweight;
  int64_t vocab, padding_idx;
  int slices;       // as EmbedSumParams
  int width;
  int zero_ctas;    // the grid's first CTAs zero rows; then one CTA a token and slice
  float scale;
};

template <typename TW, typename TO, bool VEC>
__global__ void __launch_bounds__(kFewThreads) embed_few_kernel(const EmbedFewParams p) {
  constexpr int kWarps = kFewThreads / 32, kSteps = kFewTokens / kFewThreads;
  __shared__ float part[kWarps][kSumSlice];
  __shared__ uint32_t present[kFewRows / 32];
  pdl_sync();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  TW* dw = static_cast<TW*>(p.dweight);
  if (static_cast<int>(blockIdx.x) < p.zero_ctas) {
    const float zero[8] = {};
    for (int64_t v0 = static_cast<int64_t>(blockIdx.x) * kFewRows; v0 < p.vocab; v0 += static_cast<int64_t>(p.zero_ctas) * kFewRows) {
      if (tid < kFewRows / 32) present[tid] = 0;
      __syncthreads();
      for (int i = tid; i < p.tokens; i += kFewThreads) {
        const int64_t id = load_id(p.ids, p.ids64, i), at = id - v0;
        if (at >= 0 && at < kFewRows && id != p.padding_idx) atomicOr(present + (at >> 5), 1u << (at & 31));
      }
      __syncthreads();
      for (int at = warp; at < kFewRows && v0 + at < p.vocab; at += kWarps)
        if (!((present[at >> 5] >> (at & 31)) & 1u))
          for (int slice = 0; slice < p.slices; ++slice)
            slice_store<TW, VEC>(dw + (v0 + at) * p.width, slice, lane, p.width, zero);
      __syncthreads();
    }
    return;
  }
  const int item = static_cast<int>(blockIdx.x) - p.zero_ctas, token = item / p.slices, slice = item % p.slices;
  const int64_t row = load_id(p.ids, p.ids64, token);
  if (row < 0 || row >= p.vocab || row == p.padding_idx) return;
  unsigned same[kSteps];  // this warp's tokens of the row, 32 of each step of 256
  bool before = false;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int i = s * kFewThreads + tid;
    const bool is = i < p.tokens && load_id(p.ids, p.ids64, i) == row;
    before |= is && i < token;
    same[s] = __ballot_sync(~0u, is);
  }
  if (__syncthreads_or(before)) return;  // the first token of the row sums it
  const TO* dout = static_cast<const TO*>(p.dout);
  float acc[8] = {};
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
    for (unsigned left = same[s]; left != 0;) {
      constexpr int kAtOnce = 4;
      SliceWords<TO, VEC> rows[kAtOnce];
      bool in[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        in[u] = left != 0;
        const int i = s * kFewThreads + warp * 32 + (in[u] ? __ffs(left) - 1 : 0);
        left &= left - 1;  // 0 stays 0
        if (in[u]) rows[u] = slice_load<TO, VEC>(dout + static_cast<int64_t>(i) * p.width, slice, lane, p.width);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (in[u]) {
          float f[8];
          slice_widen<TO, VEC>(rows[u], f);
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] += f[k];
        }
    }
#pragma unroll
  for (int k = 0; k < 8; ++k) part[warp][k * 32 + lane] = acc[k];
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int w = 1; w < kWarps; ++w)
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] += part[w][k * 32 + lane];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] *= p.scale;
    slice_store<TW, VEC>(dw + row * p.width, slice, lane, p.width, acc);
  }
}

}  // namespace fp8b
