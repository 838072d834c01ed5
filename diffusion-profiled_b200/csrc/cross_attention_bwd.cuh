// cross_attention_bwd.cuh — gradient of the attention of cross_attention.cuh.
//
// Two launches, each with its sums in tensor memory from beginning to end, so that no
// gradient is added to memory by several CTAs (no atomics, one order of addition):
//   * x_dq_kernel: a row tile of queries against its key tiles, 128 keys at a step.  Per
//     step S = Q K^T and dP = dO V^T, dS = P (dP - delta), dQ += dS K.  It also leaves
//     each row's -log-sum-exp and -delta for the second launch;
//   * x_dkv_kernel: a key tile against the rows that read it, 64 at a step, all heads that
//     share it among them.  The scores are formed transposed, S^T = K Q^T and
//     dP^T = V dO^T (lane = key), so that P^T and dS^T lie in tensor memory as the first
//     operands of dV += P^T dO and dK += dS^T Q.
// That is seven products a tile pair; a single launch would need five, but would add
// dQ to memory from every key tile.  Both kernels know the rows' log-sum-exp, so no
// maximum is searched and a row of scores needs no single owner: 16 softmax warps take
// 32 columns of a row each.  One warp issues the scores and dP, one the gradients.
//
// What runs side by side.  x_dq_kernel: the scores run a tile ahead into a second buffer,
// dP one tile ahead of its use as soon as the last has been read; all 16 warps work on one
// tile.  (64 keys at a step, two groups of warps by turns as in x_dkv_kernel: 257 to 279 us
// against 198 for 2 x 4096 queries of 8 heads of 128 over 4096 keys: products of 64 columns
// run at two thirds of the rate, and dQ's sum leaves tensor memory room enough without
// them.)  x_dkv_kernel, whose two sums leave room for one tile's scores and dP only: two
// buffers of 64 rows, and two groups of eight warps that take the steps by turns, so that
// one group's exponentials run during the other's products.  (One buffer of 128 rows: 298 us
// against 275.)  Both are bound by the products and the softmax by turns, at 1,040 and 1,000
// TFLOP/s of the seven products they do, 60 to 63 % of the measured peak; 13 % of the time is
// the last wave of 512 tiles on 148 SMs.
//
// delta_i = do_i . o_i from the forward's output; where the states are at most one key
// tile (SPLIT), delta_i = sum_j p_ij dp_ij in fp32 instead, without the output's rounding
// (with few keys it does not average out), P and dS go into the products as the sum of two
// values of the tensors' type, and a sequence of one key gets the exact zero that its dS
// is.  Otherwise P and dS are rounded to the type once (they are matrix operands); scores,
// dP, statistics and all sums are fp32.
//
// fp16 has too few exponents for P and dS as they are: over 4096 keys a weight is near 2^-12,
// and times a gradient of 2^-10 it would be a few multiples of 2^-24, the smallest step.  So
// both go into their products times powers of two, which are taken out of the sums again.
// P <= 1 is taken times 2^14.  |dS_ij| <= p_ij |do_i| (|v_j| + |o_i|) <= 2 |do_i| max|v|, and
// dS is taken times the power of two that brings this bound to between 2^13 and 2^14: each
// row's own in dQ, and for dK, where rows are added up, the one of the key head's largest
// |do|.  x_norms_kernel finds these norms (fp16 alone; with it 5 x 333 queries of 8 heads of
// 80 over 1021 keys take 91 us a training call, 83 without).
//
// A barrier that warps arrive on has one copy for each buffer, and the buffer is reused only
// after its phase: with one for all, a warp that is a step ahead completes a phase that
// another has not reached.
#pragma once

#include "cross_attention.cuh"

namespace fp8b {

constexpr int kXBwdWarps = 16;                      // softmax warps, two groups of eight
constexpr int kXBwdThreads = kXBwdWarps * 32 + 96;  // and loads, scores, gradients

struct XBwdParams {
  XAttnParams a;
  int row_tiles;  // row tiles of a (sequence, head group)
  int hv;         // head groups: heads / pack
  // [batch][head groups][row_tiles][2][128]: -log-sum-exp in log2 units (-inf where the row has no weight), -delta
  float* stats;
  uint32_t items;
  // x_dkv_kernel
  int q_tiles;    // row tiles that read a key head: (group / pack) * row_tiles
  int q_chunk;    // row tiles of a split; splits == 1: all of them
  int splits;
  float* part;    // [splits][2][batch][k_len][kv_heads][head_dim] (dv, dk * scale), with splits > 1
  // fp16 (x_norms_kernel): |dout|^2 of each row [batch][heads][q_len], and of each key head [batch][kv_heads][2] the largest,
  // and the largest |v|^2 of its kept keys, as the bits of a float
  float* row_norm2;
  unsigned int* max_norm2;
};

// fp16's powers of two (see above): P's, and the one for dS from the squares of the norms.
template <typename T>
constexpr bool kXScaled = std::is_same_v<T, __half>;
constexpr int kXWeightExp = 14;
__device__ __forceinline__ int x_ds_exp(float do2, float v2) {
  const float bound = 2.0f * sqrtf(do2) * sqrtf(v2);
  if (!(bound > 0.0f) || bound > 3.0e38f) return 0;  // no gradient, or no finite one
  return max(-60, min(60, kXWeightExp - (static_cast<int>(__float_as_uint(bound) >> 23) - 126)));
}
__device__ __forceinline__ float x_exp2i(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Sum of the products of eight 16-bit values.
template <typename T>
__device__ __forceinline__ float x_dot8(const uint4& x, const uint4& y) {
  const T* u = reinterpret_cast<const T*>(&x);
  const T* v = reinterpret_cast<const T*>(&y);
  float s[2] = {0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < 8; ++k) s[k & 1] = fmaf(to_f32(u[k]), to_f32(v[k]), s[k & 1]);
  return s[0] + s[1];
}

// All lanes have done what came before.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Weights and score gradients of a chunk of 32 columns, as operands over the columns they were made from.
template <typename T, bool SPLIT>
__device__ __forceinline__ void x_store_operand(uint32_t taddr, const float (&x)[32]) {
  uint32_t hi[16], lo[16];
#pragma unroll
  for (int k = 0; k < 32; k += 2) {
    if constexpr (SPLIT) split2<T>(x[k], x[k + 1], hi[k >> 1], lo[k >> 1]);
    else hi[k >> 1] = XType<T>::pack2(x[k], x[k + 1]);
  }
  tmem_st_32x32b_x16(taddr, hi);
  if constexpr (SPLIT) tmem_st_32x32b_x16(taddr + 16, lo);
}

// D += A B over `steps` (of at most MAX) 16-column steps of an operand stored by x_store_operand and a tile read across
// its rows (one elected thread).
template <bool SPLIT, int MAX>
__device__ __forceinline__ void x_products_mn(uint32_t d, uint32_t operand, uint64_t b, uint32_t idesc, int steps,
                                              uint32_t accumulate) {
#pragma unroll
  for (int k = 0; k < MAX; ++k)
    if (k < steps) {
      const uint32_t w = operand + (k >> 1) * 32 + (k & 1) * 8;
      umma_f16_ts(d, w, b + k * 128, idesc, k > 0 ? 1u : accumulate);
      if (SPLIT) umma_f16_ts(d, w + 16, b + k * 128, idesc, 1u);
    }
}

// ============================================================================ norms (fp16)
// A CTA takes kXNormRows rows of dO, and of V, of a (sequence, key head) at a time; 16 lanes a row, eight channels each,
// four rows' loads under way.
constexpr int kXNormAtOnce = 4, kXNormRows = 16 * kXNormAtOnce;
template <typename T>
__global__ void __launch_bounds__(256) x_norms_kernel(const XBwdParams p) {
  __shared__ unsigned int most[2];
  pdl_sync();
  const XAttnParams& a = p.a;
  const int lane = threadIdx.x & 15, first = threadIdx.x >> 4;
  const int64_t q_rows = static_cast<int64_t>(a.q_len) * a.group, rows = q_rows + a.k_len;
  const int64_t chunks = (rows + kXNormRows - 1) / kXNormRows, items = chunks * a.batch * a.kv_heads;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t head = item / chunks;  // of all sequences' key heads
    const int b = static_cast<int>(head / a.kv_heads), hk = static_cast<int>(head % a.kv_heads);
    const int count = x_key_count(a, x_raw_count(a, b));
    if (threadIdx.x < 2) most[threadIdx.x] = 0;
    __syncthreads();
    uint4 w[kXNormAtOnce];
    int64_t row_of[kXNormAtOnce];  // of dO: where its norm goes; of V: -1; no such row: -2
#pragma unroll
    for (int u = 0; u < kXNormAtOnce; ++u) {
      const int64_t r = item % chunks * kXNormRows + first + 16 * u;
      const bool is_q = r < q_rows;
      const int token = static_cast<int>(is_q ? r / a.group : r - q_rows), h = hk * a.group + static_cast<int>(r % a.group);
      const T* row = is_q ? static_cast<const T*>(a.dout) + b * a.sdo.batch + token * a.sdo.token + h * a.sdo.head
                          : static_cast<const T*>(a.v) + b * a.sv.batch + token * a.sv.token + hk * a.sv.head;
      const bool used = is_q || (r < rows && token < count && x_key_kept(a, b, token));
      row_of[u] = is_q ? (static_cast<int64_t>(b) * a.heads + h) * a.q_len + token : used ? -1 : -2;
      w[u] = make_uint4(0, 0, 0, 0);
      if (used && lane * 8 < a.head_dim) w[u] = *reinterpret_cast<const uint4*>(row + lane * 8);
    }
#pragma unroll
    for (int u = 0; u < kXNormAtOnce; ++u) {
      float sum = x_dot8<T>(w[u], w[u]);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);  // (within the row's 16 lanes)
      if (lane == 0 && row_of[u] > -2) {
        if (row_of[u] >= 0) p.row_norm2[row_of[u]] = sum;
        atomicMax(most + (row_of[u] >= 0 ? 0 : 1), __float_as_uint(sum));  // (not negative: as bits in the same order, NaN above all)
      }
    }
    __syncthreads();
    if (threadIdx.x < 2) atomicMax(p.max_norm2 + 2 * head + threadIdx.x, most[threadIdx.x]);
    __syncthreads();
  }
}

// ============================================================================ dQ
template <int HALVES, bool SPLIT>
struct XDqLayout {
  static constexpr int kTileBytes = HALVES * 16384;
  // Sums of dQ in tensor memory.  With two, an item's is handed out while the next item's products run; with heads of
  // more than 64 there is room for one (and items are longer).
  static constexpr int kAccs = HALVES == 1 ? 2 : 1;
  static constexpr int kDeltas = SPLIT ? 1 : kAccs;  // buffers of the rows' delta in parts
  static constexpr int kQStages = HALVES == 1 ? (SPLIT ? 4 : 3) : 1;  // Q and dO of an item
  // A key tile stays from its scores to its dQ product, two tiles later; a value tile only for its dP.
  static constexpr int kKStages = HALVES == 1 ? (SPLIT ? 3 : 4) : SPLIT ? 2 : 3;
  static constexpr int kVStages = HALVES == 1 && !SPLIT ? 3 : 2;
  static constexpr int kK = 2 * kQStages * kTileBytes;
  static constexpr int kV = kK + kKStages * kTileBytes;
  static constexpr int kWords = kV + kVStages * kTileBytes;
  static constexpr int kDelta = kWords + kXMaskSlots * 16;  // fp32 [kDeltas][2 or, with SPLIT, 4][128]
  static constexpr int kBar = kDelta + (SPLIT ? 2048 : kDeltas * 1024);
  static constexpr int kNumBars = 2 * (kQStages + kKStages + kVStages) + 18;
  static constexpr int kTail = kBar + kNumBars * 8;
  static constexpr int kSmemBytes = kTail + 16 + 1024;
};
static_assert(XDqLayout<1, true>::kSmemBytes <= 232448 && XDqLayout<2, true>::kSmemBytes <= 232448 &&
                  XDqLayout<1, false>::kSmemBytes <= 232448 && XDqLayout<2, false>::kSmemBytes <= 232448, "dq smem");
// tensor memory columns: two score buffers (dS over them), dP, dQ
constexpr uint32_t kXDqS = 0, kXDqDP = 256, kXDqAcc = 384;

struct XDqItem {
  int b, hv, tile, keys, tiles;
};
// As XItems; `ahead` is the item after the one that next() gave.
struct XDqItems {
  const XBwdParams& p;
  const XCount by;
  uint32_t i;
  XCount at;
  int keys = 0;
  __device__ __forceinline__ explicit XDqItems(const XBwdParams& q)
      : p(q), by(x_count(gridDim.x, q.row_tiles, q.hv, 1u << 30)), i(blockIdx.x),
        at(x_count(blockIdx.x, q.row_tiles, q.hv, 1u << 30)) {
    if (i < p.items) keys = x_raw_count(p.a, at.d2);
  }
  __device__ __forceinline__ bool ahead(XDqItem& t) const {
    t.tile = at.d0;
    t.hv = at.d1;
    t.b = at.d2;
    t.keys = x_key_count(p.a, keys);
    t.tiles = (t.keys + kXTile - 1) / kXTile;
    return i < p.items;
  }
  __device__ __forceinline__ bool next(XDqItem& t) {
    if (!ahead(t)) return false;
    i += gridDim.x;
    x_advance(at, by, p.row_tiles, p.hv, 1 << 30);
    if (i < p.items) keys = x_raw_count(p.a, at.d2);
    return true;
  }
};

template <typename T, int HALVES, bool SPLIT>
__global__ void __launch_bounds__(kXBwdThreads, 1)
    x_dq_kernel(const XBwdParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap do_map,
                const __grid_constant__ CUtensorMap dq_map) {
  using Ly = XDqLayout<HALVES, SPLIT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint4* words = reinterpret_cast<uint4*>(smem + Ly::kWords);
  float* delta_part = reinterpret_cast<float*>(smem + Ly::kDelta);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + Ly::kBar);
  uint64_t* q_empty = q_full + Ly::kQStages;
  uint64_t* k_full = q_empty + Ly::kQStages;
  uint64_t* k_empty = k_full + Ly::kKStages;
  uint64_t* v_full = k_empty + Ly::kKStages;
  uint64_t* v_empty = v_full + Ly::kVStages;
  uint64_t* s_full = v_empty + Ly::kVStages;  // [2], by score buffer
  uint64_t* s_free = s_full + 2;              // [2]: its dS has been multiplied
  uint64_t* dp_full = s_free + 2;
  uint64_t* dp_free = dp_full + 1;
  uint64_t* ds_full = dp_free + 1;            // [2], by score buffer: a warp may be a tile ahead of another
  uint64_t* acc_full = ds_full + 2;  // [2], by sum
  uint64_t* acc_free = acc_full + 2;
  uint64_t* staged = acc_free + 2;
  uint64_t* delta_full = staged + 2;   // [2], by buffer of delta
  uint64_t* drained = delta_full + 2;  // [2], by issuing warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Ly::kTail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < Ly::kQStages; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
    }
    for (int i = 0; i < Ly::kKStages; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
    }
    for (int i = 0; i < Ly::kVStages; ++i) {
      mbar_init(v_full + i, 1);
      mbar_init(v_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 2);  // the products' commit, and the issuing thread (keep bits)
      mbar_init(s_free + i, 1);
      mbar_init(ds_full + i, kXBwdWarps);
      mbar_init(drained + i, 1);
      mbar_init(acc_full + i, 1);
      mbar_init(acc_free + i, kXBwdWarps);
      mbar_init(staged + i, kXBwdWarps);
      mbar_init(delta_full + i, SPLIT ? kXBwdWarps : 8);
    }
    mbar_init(dp_full, 2);  // the products' commit, and the issuing warp (rows of K zeroed)
    mbar_init(dp_free, kXBwdWarps);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kXBwdWarps) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  const XAttnParams& a = p.a;
  const bool masked = a.key_mask != nullptr;
  const int ksteps = (a.head_dim + 15) >> 4;
  const uint32_t s_base = smem_u32(smem);
  const auto wait = [&](uint64_t* bar, uint32_t phase, int what) {
    return warp_wait(bar, phase & 1, abort_flag, a.err, kErrXDq + what);
  };

  if (warp == kXBwdWarps) {
    // ------------------------------------------------------------ loads
    const uint32_t q_bytes = static_cast<uint32_t>(a.tile_tokens * a.pack) * 128u * HALVES;
    uint32_t n_item = 0, g = 0, n_k = 0, n_v = 0;  // n_k, n_v: copies started
    bool ok = true;
    XDqItems items(p);
    XDqItem t;
    while (ok && items.next(t)) {
      if (t.tiles == 0) continue;
      const int qs = n_item % Ly::kQStages;
      ok = wait(q_empty + qs, (n_item / Ly::kQStages) ^ 1, kWaitQFree);
      if (!ok) break;
      if (lane == 0) {
        uint8_t* dst = smem + 2 * qs * Ly::kTileBytes;
        mbar_arrive_expect_tx(q_full + qs, 2 * q_bytes);
        for (int hf = 0; hf < HALVES; ++hf) {
          tma_load_4d(dst + hf * 16384, &q_map, q_full + qs, hf * 64, t.hv * a.pack, t.tile * a.tile_tokens, t.b);
          tma_load_4d(dst + Ly::kTileBytes + hf * 16384, &do_map, q_full + qs, hf * 64, t.hv * a.pack,
                      t.tile * a.tile_tokens, t.b);
        }
      }
      ++n_item;
      const int hk = t.hv * a.pack / a.group;
      for (int j = 0; j < t.tiles; ++j, ++g) {
        if (masked || (j + 1) * kXTile > t.keys) {
          const uint4 w = x_keep_words(a, t.b, j * kXTile, t.keys, lane);
          if (lane == 0) words[g % kXMaskSlots] = w;
        }
        const int ks = g % Ly::kKStages, vs = g % Ly::kVStages;
        ok = wait(k_empty + ks, (g / Ly::kKStages) ^ 1, kWaitKFree);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(k_full + ks, Ly::kTileBytes);
          for (int hf = 0; hf < HALVES; ++hf)
            tma_load_4d(smem + Ly::kK + ks * Ly::kTileBytes + hf * 16384, &k_map, k_full + ks, hf * 64, hk, j * kXTile, t.b);
        }
        ++n_k;
        ok = wait(v_empty + vs, (g / Ly::kVStages) ^ 1, kWaitVFree);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(v_full + vs, Ly::kTileBytes);
          for (int hf = 0; hf < HALVES; ++hf)
            tma_load_4d(smem + Ly::kV + vs * Ly::kTileBytes + hf * 16384, &v_map, v_full + vs, hf * 64, hk, j * kXTile, t.b);
        }
        ++n_v;
      }
    }
    if (!ok && lane == 0) {  // copies still in flight land before the CTA leaves
      volatile int never = 0;
      const auto drain = [&](uint64_t* full, uint32_t stages, uint32_t n) {
        for (uint32_t k = n > stages ? n - stages : 0; k < n; ++k)
          mbar_wait(full + k % stages, (k / stages) & 1, &never, a.err, kErrXDq + kWaitDrain);
      };
      drain(q_full, Ly::kQStages, n_item);
      drain(k_full, Ly::kKStages, n_k);
      drain(v_full, Ly::kVStages, n_v);
    }
  } else if (warp == kXBwdWarps + 1) {
    // ------------------------------------------------------------ products S = Q K^T, dP = dO V^T
    uint32_t n_item = 0, g = 0;
    bool ok = true;
    XDqItems items(p);
    XDqItem t;
    while (ok && items.next(t)) {
      if (t.tiles == 0) continue;
      const int qs = n_item % Ly::kQStages;
      ok = wait(q_full + qs, n_item / Ly::kQStages, kWaitQ);
      const uint64_t sq = k_major_desc(s_base + 2 * qs * Ly::kTileBytes);
      const uint64_t sdo = k_major_desc(s_base + (2 * qs + 1) * Ly::kTileBytes);
      for (int j = 0; j < t.tiles && ok; ++j, ++g) {
        const int ks = g % Ly::kKStages, vs = g % Ly::kVStages, buf = g & 1;
        const uint32_t idesc = x_idesc<T>(x_chunks(t.keys, j) * 32, 0, 0);
        const bool bits = masked || (j + 1) * kXTile > t.keys;
        uint8_t* sk = smem + Ly::kK + ks * Ly::kTileBytes;
        uint8_t* sv = smem + Ly::kV + vs * Ly::kTileBytes;
        if (!(ok = wait(k_full + ks, g / Ly::kKStages, kWaitK))) break;
        uint4 w = make_uint4(~0u, ~0u, ~0u, ~0u);
        if (bits) w = words[g % kXMaskSlots];
        const bool holes = (w.x & w.y & w.z & w.w) != 0xffffffffu;
        if (g >= 2 && !(ok = wait(s_free + buf, (g >> 1) ^ 1, kWaitSFree))) break;
        tc_fence_after();
        if (elect_one()) {
          products_k_major(tmem + kXDqS + buf * 128, sq, k_major_desc(smem_u32(sk)), idesc, ksteps);
          umma_commit(s_full + buf);
          mbar_arrive(s_full + buf);
        }
        __syncwarp();
        // Keys that are not kept: K with zeros for dQ, where the zeros of dS would not keep an infinity out (what the scores
        // read there is replaced), V for dP, so that dS gets them.
        if (holes) x_zero_rows<HALVES>(sk, w, x_chunks(t.keys, j) * 32, lane);
        if (!(ok = wait(v_full + vs, g / Ly::kVStages, kWaitV))) break;
        if (holes) x_zero_rows<HALVES>(sv, w, x_chunks(t.keys, j) * 32, lane);
        if (g >= 1 && !(ok = wait(dp_free, g ^ 1, kWaitDPFree))) break;
        tc_fence_after();
        if (elect_one()) {
          products_k_major(tmem + kXDqDP, sdo, k_major_desc(smem_u32(sv)), idesc, ksteps);
          umma_commit(v_empty + vs);
          umma_commit(dp_full);
          mbar_arrive(dp_full);
        }
        __syncwarp();
      }
      ++n_item;
    }
    if (!ok && elect_one()) {  // the products in flight end before the tensor memory is freed
      volatile int never = 0;
      umma_commit(drained);
      mbar_wait(drained, 0, &never, a.err, kErrXDq + kWaitDrain);
    }
  } else if (warp == kXBwdWarps + 2) {
    // ------------------------------------------------------------ products dQ += dS K
    const uint32_t idesc = x_idesc<T>(ksteps * 16, 0, 1);
    uint32_t n_item = 0, g = 0;
    bool ok = true;
    XDqItems items(p);
    XDqItem t;
    while (ok && items.next(t)) {
      if (t.tiles == 0) continue;
      for (int j = 0; j < t.tiles; ++j, ++g) {
        const int ks = g % Ly::kKStages, buf = g & 1, steps = 2 * x_chunks(t.keys, j);
        ok = wait(k_full + ks, g / Ly::kKStages, kWaitK) && wait(ds_full + buf, g >> 1, kWaitP);
        if (ok && j == 0 && n_item >= Ly::kAccs)  // the last dQ summed here has been read
          ok = wait(acc_free + n_item % Ly::kAccs, (n_item / Ly::kAccs) ^ 1, kWaitAccFree);
        if (!ok) break;
        const uint64_t sk = mn_major_desc(s_base + Ly::kK + ks * Ly::kTileBytes);
        tc_fence_after();
        if (elect_one()) {
          x_products_mn<SPLIT, 8>(tmem + kXDqAcc + n_item % Ly::kAccs * 64, tmem + kXDqS + buf * 128, sk, idesc, steps, j > 0 ? 1u : 0u);
          umma_commit(s_free + buf);
          umma_commit(k_empty + ks);
          if (j == t.tiles - 1) umma_commit(acc_full + n_item % Ly::kAccs);
        }
        __syncwarp();
      }
      ++n_item;
    }
    if (!ok && elect_one()) {
      volatile int never = 0;
      umma_commit(drained + 1);
      mbar_wait(drained + 1, 0, &never, a.err, kErrXDq + kWaitDrain);
    }
  } else {
    // ------------------------------------------------------------ dS: thread = row, the 32 columns of chunk wq
    const int wq = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c2 = a.scale * 1.4426950408889634f;
    const uint64_t c22 = pair2(c2, c2);
    const int rows = a.tile_tokens * a.pack;
    const int my_token = row / a.pack, my_head = row % a.pack;
    // This row's log-sum-exp and, in the first two chunks' warps, half of the channels of its output, for the item to
    // come: asked for while the products of the item before still run.  (With heads of 128 the output is read when the
    // item begins: the registers for it are not there, and items are longer.)
    uint4 o_row[4];
    float lse = -INFINITY;
    float do2 = 0.0f, v2 = 0.0f;  // fp16: the squares of this row's |dO| and of its keys' largest |V|
    const auto fetch = [&](const XDqItems& items) {
      XDqItem t;
      const bool exists = items.ahead(t);
      const int token = t.tile * a.tile_tokens + my_token, head = t.hv * a.pack + my_head;
      const bool live = exists && t.tiles > 0 && row < rows && token < a.q_len;
      if (!SPLIT && HALVES == 1 && wq < 2) {
        const T* o = static_cast<const T*>(a.o_in) + t.b * a.so.batch + token * a.so.token + head * a.so.head;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = wq * 32 + 8 * u;
          o_row[u] = live && c < a.head_dim ? *reinterpret_cast<const uint4*>(o + c) : make_uint4(0, 0, 0, 0);
        }
      }
      const int64_t r_index = (static_cast<int64_t>(t.b) * a.heads + head) * a.q_len + token;
      lse = live ? a.lse[r_index] : -INFINITY;
      if constexpr (kXScaled<T>) {
        do2 = live ? p.row_norm2[r_index] : 0.0f;
        v2 = live ? __uint_as_float(p.max_norm2[2 * (static_cast<int64_t>(t.b) * a.kv_heads + head / a.group) + 1]) : 0.0f;
      }
    };
    uint32_t n_item = 0, g = 0;
    int stored = -1;  // Q stage whose gradient is on its way out
    const auto release_stored = [&]() {
      if (stored >= 0 && tid == 0) {
        bulk_wait_group_read<0>();
        mbar_arrive(q_empty + stored);
      }
      stored = -1;
    };
    // The gradient of item n, from its sum by way of Q's tile, which every product of the item has read by then: a quarter
    // of the channels each.
    struct Done {
      uint32_t n;
      int b, hv, tile;
      bool dead;
      float scale;  // fp16: of the sum
    };
    const auto hand_out = [&](const Done& w) {
      const uint32_t acc = w.n % Ly::kAccs, phase = w.n / Ly::kAccs;
      const int qs = w.n % Ly::kQStages;
      const float f = kXScaled<T> ? w.scale : a.scale;
      uint8_t* stage = smem + 2 * qs * Ly::kTileBytes;
      release_stored();
      if (!wait(acc_full + acc, phase, kWaitAcc)) return false;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < HALVES; ++c) {
        const int col = (wq * HALVES + c) * 16;
        uint32_t o[16];
        tmem_read(t_lane + kXDqAcc + acc * 64 + col, o);
        uint32_t pk[8];
#pragma unroll
        for (int k = 0; k < 16; k += 2)
          pk[k >> 1] = w.dead ? 0u : XType<T>::pack2(__uint_as_float(o[k]) * f, __uint_as_float(o[k + 1]) * f);
        uint8_t* half = stage + (col >> 6) * 16384;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          st_shared_v4(half + swizzle128_offset(row, ((col & 63) >> 3) + u), pk[4 * u], pk[4 * u + 1], pk[4 * u + 2],
                       pk[4 * u + 3]);
      }
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(staged + acc);
        mbar_arrive(acc_free + acc);
      }
      bool ok = true;
      if (tid == 0) {
        ok = mbar_wait(staged + acc, phase & 1, abort_flag, a.err, kErrXDq + kWaitStaged);
        if (ok) {
          for (int hf = 0; hf < HALVES; ++hf)
            tma_store_4d(&dq_map, stage + hf * 16384, hf * 64, w.hv * a.pack, w.tile * a.tile_tokens, w.b);
          bulk_commit_group();
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (ok) stored = qs;
      if (Ly::kQStages == 1) release_stored();
      return ok;
    };
    Done done{};  // not handed out yet, with two sums
    bool any_done = false, ok = true;
    XDqItems items(p);
    XDqItem t;
    fetch(items);
    while (ok && items.next(t)) {
      const int token = t.tile * a.tile_tokens + my_token, head = t.hv * a.pack + my_head;
      float* stat = p.stats + ((static_cast<int64_t>(t.b) * p.hv + t.hv) * p.row_tiles + t.tile) * (2 * kXTile) + row;
      if (t.tiles == 0) {  // no keys
        if (wq == 0) {
          stat[0] = -INFINITY;
          stat[kXTile] = 0.0f;
          if (row < rows && token < a.q_len) {
            T* o = static_cast<T*>(a.dq) + t.b * a.sdq.batch + token * a.sdq.token + head * a.sdq.head;
            for (int c = 0; c < a.head_dim; c += 8) *reinterpret_cast<uint4*>(o + c) = make_uint4(0, 0, 0, 0);
          }
        }
        fetch(items);
        continue;
      }
      const int qs = n_item % Ly::kQStages;
      uint8_t* stage = smem + 2 * qs * Ly::kTileBytes;
      const bool dead = lse == -INFINITY;  // no such row, or no kept key
      const float neg_lse = dead ? -INFINITY : -lse * 1.4426950408889634f;
      const int ds_exp = kXScaled<T> ? x_ds_exp(do2, v2) : 0;
      float neg_delta = 0.0f;
      float* parts = delta_part + n_item % Ly::kDeltas * (2 * kXTile);
      // (Half of the warps arrive and all wait.  An item of one key tile may let those that arrive go on to the next item's
      // delta before the others have seen this one's; the one after that they reach only behind dP of the next item, which
      // waits for all to have read dP of this one: two copies.)
      uint64_t* const delta_here = delta_full + n_item % Ly::kDeltas;
      if (!SPLIT && wq < 2) {  // delta = do . o, half of the channels each
        ok = wait(q_full + qs, n_item / Ly::kQStages, kWaitQ);
        if (!ok) break;
        float part = 0.0f;
        const T* o = static_cast<const T*>(a.o_in) + t.b * a.so.batch + token * a.so.token + head * a.so.head;
#pragma unroll
        for (int u = 0; u < HALVES * 4; ++u) {
          const int c = wq * HALVES * 4 + u;  // 16-byte chunk of the row
          uint4 v = make_uint4(0, 0, 0, 0);
          if constexpr (HALVES == 1) {
            v = o_row[u];
          } else if (!dead && c * 8 < a.head_dim) {
            v = *reinterpret_cast<const uint4*>(o + c * 8);
          }
          part -= x_dot8<T>(v, ld_shared_v4(stage + Ly::kTileBytes + (c >> 3) * 16384 + swizzle128_offset(row, c & 7)));
        }
        parts[wq * kXTile + row] = part;
        warp_arrive(delta_here);
      }
      // this row's delta, from its parts, and the statistics that the second launch needs
      const auto join_delta = [&]() {
        if (!wait(delta_here, n_item / Ly::kDeltas, kWaitDelta)) return false;
        neg_delta = parts[row] + parts[kXTile + row];
        if (SPLIT) neg_delta += parts[2 * kXTile + row] + parts[3 * kXTile + row];
        if (SPLIT && kXScaled<T>) neg_delta *= x_exp2i(-ds_exp);  // (summed with the weights that dS is made from)
        if (dead) neg_delta = 0.0f;
        if (wq == 0) {
          stat[0] = neg_lse;
          stat[kXTile] = neg_delta;
        }
        return true;
      };
      if (!SPLIT) {
        ok = join_delta();
        if (!ok) break;
      }
      const float nl = kXScaled<T> ? neg_lse + static_cast<float>(ds_exp) : neg_lse;
      const uint64_t nl2 = pair2(nl, nl);
      for (int j = 0; j < t.tiles; ++j, ++g) {
        const uint32_t t_s = t_lane + kXDqS + (g & 1) * 128 + wq * 32;
        const bool some = wq < x_chunks(t.keys, j);  // the chunk holds keys
        ok = wait(s_full + (g & 1), g >> 1, kWaitS);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[32];
        bool single = false;  // one kept key: its weight is 1 whatever its score, and no gradient goes through it
        if (some) {
          tmem_read(t_s, s);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float x0, x1;
            unpair2(fma2(pair2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), c22, nl2), x0, x1);
            s[k] = __float_as_uint(ex2(x0));
            s[k + 1] = __float_as_uint(ex2(x1));
          }
          if (masked || (j + 1) * kXTile > t.keys) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(words + g % kXMaskSlots)[wq];
            if (SPLIT) {
              const uint4 all = words[g % kXMaskSlots];
              single = __popc(all.x) + __popc(all.y) + __popc(all.z) + __popc(all.w) == 1;
            }
            if (w != ~0u) {
#pragma unroll
              for (int k = 0; k < 32; ++k) s[k] = (w >> k) & 1u ? s[k] : 0u;
            }
          }
        }
        if (Ly::kAccs > 1) release_stored();
        ok = wait(dp_full, g, kWaitDP);
        if (!ok) break;
        tc_fence_after();
        if constexpr (SPLIT) {  // delta = sum p dP, a chunk of it by each warp of these rows
          float s0 = 0.0f, s1 = 0.0f;
          if (some) {
            uint64_t sum = pair2(0.0f, 0.0f);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t dp[16];
              tmem_read(t_lane + kXDqDP + wq * 32 + h * 16, dp);
#pragma unroll
              for (int k = 0; k < 16; k += 2)
                sum = fma2(pair2(__uint_as_float(s[16 * h + k]), __uint_as_float(s[16 * h + k + 1])),
                           pair2(__uint_as_float(dp[k]), __uint_as_float(dp[k + 1])), sum);
            }
            unpair2(sum, s0, s1);
          }
          parts[wq * kXTile + row] = -(s0 + s1);
          warp_arrive(delta_here);
          ok = join_delta();
          if (!ok) break;
        }
        const uint64_t nd2 = pair2(neg_delta, neg_delta);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t dp[16];
          if (some) tmem_read(t_lane + kXDqDP + wq * 32 + h * 16, dp);
          if (h == 1) {
            tc_fence_before();
            warp_arrive(dp_free);
          }
          if (some) {
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              const uint64_t d = add2(pair2(__uint_as_float(dp[k]), __uint_as_float(dp[k + 1])), nd2);
              float x0, x1;
              unpair2(mul2(pair2(__uint_as_float(s[16 * h + k]), __uint_as_float(s[16 * h + k + 1])), d), x0, x1);
              // in the place of the weights
              if constexpr (SPLIT) {
                if (single) x0 = x1 = 0.0f;
                split2<T>(x0, x1, s[16 * h + k], s[16 * h + k + 1]);
              } else {
                s[16 * h + k] = XType<T>::pack2(x0, x1);
              }
            }
          }
        }
        if (some) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            hi[k] = s[2 * k];
            lo[k] = s[2 * k + 1];
          }
          tmem_st_32x32b_x16(t_s, hi);
          if constexpr (SPLIT) tmem_st_32x32b_x16(t_s + 16, lo);
          tmem_st_wait();
        }
        tc_fence_before();
        warp_arrive(ds_full + (g & 1));
      }
      if (!ok) break;
      fetch(items);
      const Done now{n_item, t.b, t.hv, t.tile, dead, kXScaled<T> ? a.scale * x_exp2i(-ds_exp) : 0.0f};
      if (Ly::kAccs == 1 || any_done) ok = hand_out(Ly::kAccs == 1 ? now : done);
      done = now;
      any_done = true;
      ++n_item;
    }
    if (ok && Ly::kAccs > 1 && any_done) hand_out(done);
    if (tid == 0) bulk_wait_group<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kXBwdWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ============================================================================ dK, dV
template <int HALVES>
struct XDkvLayout {
  static constexpr int kTileBytes = HALVES * 16384;
  static constexpr int kKVStages = HALVES == 1 ? 2 : 1;  // K and V of an item
  static constexpr int kEntries = HALVES == 1 ? 8 : 4;   // Q and dO tiles in turn
  static constexpr int kQ = 2 * kKVStages * kTileBytes;
  static constexpr int kStats = kQ + kEntries * kTileBytes;  // fp32 [kEntries / 2][2][128]
  static constexpr int kWords = kStats + kEntries / 2 * 1024;
  static constexpr int kBar = kWords + 2 * kKVStages * 16;
  static constexpr int kNumBars = 2 * kKVStages + 2 * kEntries + 14;
  static constexpr int kTail = kBar + kNumBars * 8;
  static constexpr int kSmemBytes = kTail + 16 + 1024;
};
static_assert(XDkvLayout<1>::kSmemBytes <= 232448 && XDkvLayout<2>::kSmemBytes <= 232448, "dkv smem");
// tensor memory columns: two buffers of S^T (P^T over it) and of dP^T (dS^T over it), dV, dK
constexpr uint32_t kXDkvS = 0, kXDkvDP = 128, kXDkvV = 256;

struct XDkvItem {
  int b, hk, tile, split, keys, j0, j1;  // row tiles [j0, j1) of the key head; none where the tile has no keys
};
struct XDkvItems {
  const XBwdParams& p;
  const int tiles;
  const XCount by;
  uint32_t i;
  XCount at;
  int keys = 0;
  __device__ __forceinline__ explicit XDkvItems(const XBwdParams& q)
      : p(q), tiles((q.a.k_len + kXTile - 1) / kXTile), by(x_count(gridDim.x, tiles, q.splits, q.a.kv_heads)),
        i(blockIdx.x), at(x_count(blockIdx.x, tiles, q.splits, q.a.kv_heads)) {
    if (i < p.items) keys = x_raw_count(p.a, at.d3);
  }
  __device__ __forceinline__ bool next(XDkvItem& t) {
    if (i >= p.items) return false;
    t.tile = at.d0;
    t.split = at.d1;
    t.hk = at.d2;
    t.b = at.d3;
    t.keys = x_key_count(p.a, keys);
    t.j0 = min(p.q_tiles, t.split * p.q_chunk);
    t.j1 = t.tile * kXTile < t.keys ? min(p.q_tiles, t.j0 + p.q_chunk) : t.j0;
    i += gridDim.x;
    x_advance(at, by, tiles, p.splits, p.a.kv_heads);
    if (i < p.items) keys = x_raw_count(p.a, at.d3);
    return true;
  }
};

// 64-row steps of row tile `tile` of a head group.
__device__ __forceinline__ int x_row_steps(const XAttnParams& a, int tile) {
  return (min(a.tile_tokens, a.q_len - tile * a.tile_tokens) * a.pack + 63) >> 6;
}

template <typename T, int HALVES, bool SPLIT>
__global__ void __launch_bounds__(kXBwdThreads, 1)
    x_dkv_kernel(const XBwdParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap do_map,
                 const __grid_constant__ CUtensorMap dk_map, const __grid_constant__ CUtensorMap dv_map) {
  using Ly = XDkvLayout<HALVES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* stats = reinterpret_cast<float*>(smem + Ly::kStats);
  uint4* words = reinterpret_cast<uint4*>(smem + Ly::kWords);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + Ly::kBar);
  uint64_t* kv_empty = kv_full + Ly::kKVStages;
  uint64_t* q_full = kv_empty + Ly::kKVStages;
  uint64_t* q_empty = q_full + Ly::kEntries;
  // [2], by buffer
  uint64_t* s_full = q_empty + Ly::kEntries;
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_full = dp_full + 2;  // P^T and dS^T are there
  uint64_t* ds_free = ds_full + 2;  // and have been multiplied
  uint64_t* staged = ds_free + 2;   // [2], by group
  uint64_t* drained = staged + 2;   // [2], by issuing warp
  uint64_t* acc_full = drained + 2;
  uint64_t* acc_free = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Ly::kTail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const XAttnParams& a = p.a;
  const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
  const int rows = a.tile_tokens * a.pack;
  if (tid == 0) {
    for (int i = 0; i < Ly::kKVStages; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 2);
    }
    for (int i = 0; i < Ly::kEntries; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);  // by the dK or dV products, before which S^T and dP^T were done
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 2);  // the products' commit, and the issuing thread (keep bits)
      mbar_init(dp_full + i, 1);
      mbar_init(ds_full + i, 8);
      mbar_init(ds_free + i, 1);
      mbar_init(staged + i, 8);
      mbar_init(drained + i, 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_free, kXBwdWarps);
    *abort_flag = 0;
    fence_barrier_init();
  }
  // rows that no copy fills (128 is not a multiple of `pack`) are zero: they are summed over
  for (int c = tid; c < (kXTile - rows) * 8 * HALVES * Ly::kEntries; c += kXBwdThreads) {
    const int r = rows + c / 8 % (kXTile - rows), tile = c / 8 / (kXTile - rows);
    *reinterpret_cast<uint4*>(smem + Ly::kQ + tile * 16384 + r * 128 + c % 8 * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  if (warp == kXBwdWarps) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  const int ksteps = (a.head_dim + 15) >> 4;
  const uint32_t s_base = smem_u32(smem);
  const auto wait = [&](uint64_t* bar, uint32_t phase, int what) {
    return warp_wait(bar, phase & 1, abort_flag, a.err, kErrXDkv + what);
  };

  if (warp == kXBwdWarps) {
    // ------------------------------------------------------------ loads
    const uint32_t q_bytes = static_cast<uint32_t>(rows) * 128u * HALVES;
    const int per_key_head = a.group / a.pack;  // head groups that read a key head (1 where all are packed)
    uint32_t e = 0, n_item = 0;  // copies started
    bool ok = true;
    XDkvItems items(p);
    XDkvItem t;
    while (ok && items.next(t)) {
      if (t.j0 >= t.j1) continue;
      const int ks = n_item % Ly::kKVStages;
      const uint4 w = x_keep_words(a, t.b, t.tile * kXTile, t.keys, lane);
      ok = wait(kv_empty + ks, (n_item / Ly::kKVStages) ^ 1, kWaitKFree);
      if (!ok) break;
      if (lane == 0) {
        words[n_item % (2 * Ly::kKVStages)] = w;
        uint8_t* dst = smem + 2 * ks * Ly::kTileBytes;
        mbar_arrive_expect_tx(kv_full + ks, 2 * Ly::kTileBytes);
        for (int hf = 0; hf < HALVES; ++hf) {
          tma_load_4d(dst + hf * 16384, &k_map, kv_full + ks, hf * 64, t.hk, t.tile * kXTile, t.b);
          tma_load_4d(dst + Ly::kTileBytes + hf * 16384, &v_map, kv_full + ks, hf * 64, t.hk, t.tile * kXTile, t.b);
        }
      }
      ++n_item;
      for (int j = t.j0; j < t.j1 && ok; ++j) {
        const int h = t.hk * per_key_head + j / p.row_tiles, tile = j % p.row_tiles;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          const int slot = e % Ly::kEntries;
          ok = wait(q_empty + slot, (e / Ly::kEntries) ^ 1, kWaitQFree);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(q_full + slot, q_bytes + (which == 0 ? 1024u : 0u));
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_4d(smem + Ly::kQ + slot * Ly::kTileBytes + hf * 16384, which ? &do_map : &q_map, q_full + slot,
                          hf * 64, h * a.pack, tile * a.tile_tokens, t.b);
            if (which == 0)
              bulk_load_1d(stats + (slot >> 1) * 2 * kXTile,
                           p.stats + ((static_cast<int64_t>(t.b) * p.hv + h) * p.row_tiles + tile) * (2 * kXTile), 1024,
                           q_full + slot);
          }
          ++e;
        }
      }
    }
    if (!ok && lane == 0) {  // copies still in flight land before the CTA leaves
      volatile int never = 0;
      const auto drain = [&](uint64_t* full, uint32_t stages, uint32_t n) {
        for (uint32_t k = n > stages ? n - stages : 0; k < n; ++k)
          mbar_wait(full + k % stages, (k / stages) & 1, &never, a.err, kErrXDkv + kWaitDrain);
      };
      drain(q_full, Ly::kEntries, e);
      drain(kv_full, Ly::kKVStages, n_item);
    }
  } else if (warp == kXBwdWarps + 1) {
    // ------------------------------------------------------------ products S^T = K Q^T, dP^T = V dO^T
    const uint32_t idesc = x_idesc<T>(64, 0, 0);
    uint32_t n_item = 0, g = 0, n = 0;  // items, row tiles, 64-row steps
    bool ok = true;
    XDkvItems items(p);
    XDkvItem t;
    while (ok && items.next(t)) {
      if (t.j0 >= t.j1) continue;
      const int ks = n_item % Ly::kKVStages;
      ok = wait(kv_full + ks, n_item / Ly::kKVStages, kWaitK);
      if (!ok) break;
      // (What lies at a key that is not kept reaches that key's lane alone, whose gradients are zeroed at the end.)
      const uint64_t sk = k_major_desc(s_base + 2 * ks * Ly::kTileBytes);
      const uint64_t sv = k_major_desc(s_base + (2 * ks + 1) * Ly::kTileBytes);
      for (int j = t.j0; j < t.j1 && ok; ++j, ++g) {
        const uint32_t eq = 2 * g % Ly::kEntries, phase = 2 * g / Ly::kEntries;
        const int steps = x_row_steps(a, j % p.row_tiles);
        for (int u = 0; u < steps; ++u, ++n) {
          const int buf = n & 1;
          if (u == 0) ok = wait(q_full + eq, phase, kWaitQ);
          if (ok && n >= 2) ok = wait(ds_free + buf, (n >> 1) ^ 1, kWaitSFree);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            products_k_major(tmem + kXDkvS + buf * 64, sk, k_major_desc(s_base + Ly::kQ + eq * Ly::kTileBytes + u * 8192), idesc,
                             ksteps);
            umma_commit(s_full + buf);
            mbar_arrive(s_full + buf);
          }
          __syncwarp();
          if (u == 0 && !(ok = wait(q_full + eq + 1, phase, kWaitV))) break;
          tc_fence_after();
          if (elect_one()) {
            products_k_major(tmem + kXDkvDP + buf * 64, sv,
                             k_major_desc(s_base + Ly::kQ + (eq + 1) * Ly::kTileBytes + u * 8192), idesc, ksteps);
            umma_commit(dp_full + buf);
          }
          __syncwarp();
        }
      }
      ++n_item;
    }
    if (!ok && elect_one()) {  // the products in flight end before the tensor memory is freed
      volatile int never = 0;
      umma_commit(drained);
      mbar_wait(drained, 0, &never, a.err, kErrXDkv + kWaitDrain);
    }
  } else if (warp == kXBwdWarps + 2) {
    // ------------------------------------------------------------ products dV += P^T dO, dK += dS^T Q
    const uint32_t idesc = x_idesc<T>(ksteps * 16, 0, 1);
    uint32_t n_item = 0, g = 0, n = 0;
    bool ok = true;
    XDkvItems items(p);
    XDkvItem t;
    while (ok && items.next(t)) {
      if (t.j0 >= t.j1) continue;
      for (int j = t.j0; j < t.j1 && ok; ++j, ++g) {
        const uint32_t eq = 2 * g % Ly::kEntries, phase = 2 * g / Ly::kEntries;
        const int steps = x_row_steps(a, j % p.row_tiles);
        for (int u = 0; u < steps; ++u, ++n) {
          const int buf = n & 1;
          if (u == 0) ok = wait(q_full + eq, phase, kWaitQ) && wait(q_full + eq + 1, phase, kWaitV);
          ok = ok && wait(ds_full + buf, n >> 1, kWaitP);
          if (ok && j == t.j0 && u == 0 && n_item > 0) ok = wait(acc_free, n_item ^ 1, kWaitAccFree);  // the last item's sums have been read
          if (!ok) break;
          const uint64_t sq = mn_major_desc(s_base + Ly::kQ + eq * Ly::kTileBytes + u * 8192);
          const uint64_t sdo = mn_major_desc(s_base + Ly::kQ + (eq + 1) * Ly::kTileBytes + u * 8192);
          const uint32_t later = j > t.j0 || u > 0 ? 1u : 0u;
          tc_fence_after();
          if (elect_one()) {
            x_products_mn<SPLIT, 4>(tmem + kXDkvV, tmem + kXDkvS + buf * 64, sdo, idesc, 4, later);
            if (u == steps - 1) umma_commit(q_empty + eq + 1);
            x_products_mn<SPLIT, 4>(tmem + kXDkvV + HALVES * 64, tmem + kXDkvDP + buf * 64, sq, idesc, 4, later);
            if (u == steps - 1) umma_commit(q_empty + eq);
            umma_commit(ds_free + buf);
            if (j == t.j1 - 1 && u == steps - 1) umma_commit(acc_full);
          }
          __syncwarp();
        }
      }
      ++n_item;
    }
    if (!ok && elect_one()) {
      volatile int never = 0;
      umma_commit(drained + 1);
      mbar_wait(drained + 1, 0, &never, a.err, kErrXDkv + kWaitDrain);
    }
  } else {
    // ------------------------------------------------------------ P^T, dS^T: thread = key and 32 rows, the steps of group gp
    const int gp = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3, key = quad * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t t_s = t_lane + kXDkvS + gp * 64 + half * 32, t_dp = t_s + (kXDkvDP - kXDkvS);  // a group's steps use one buffer
    const float c2 = a.scale * 1.4426950408889634f;
    const uint64_t c22 = pair2(c2, c2);
    const bool hands_out = (warp & 7) == 0 && lane == 0;  // of dV (group 0) or dK (group 1)
    uint32_t n_item = 0, g = 0, n = 0;
    int stored = -1;  // K / V stage whose gradient is on its way out
    const auto release_stored = [&]() {
      if (stored >= 0 && hands_out) {
        bulk_wait_group_read<0>();
        mbar_arrive(kv_empty + stored);
      }
      stored = -1;
    };
    bool ok = true;
    XDkvItems items(p);
    XDkvItem t;
    while (ok && items.next(t)) {
      const int j_key = t.tile * kXTile + key;
      const auto part = [&](int c) {  // this key's row of the split's partial sums
        return p.part + ((((static_cast<int64_t>(t.split) * 2 + gp) * a.batch + t.b) * a.k_len + j_key) * a.kv_heads + t.hk) *
                            a.head_dim + c;
      };
      if (t.j0 >= t.j1) {  // no keys in this tile (or no rows in this split)
        if (j_key < a.k_len && half == 0) {
          T* grad = gp ? static_cast<T*>(a.dk) + t.b * a.sdk.batch + j_key * a.sdk.token + t.hk * a.sdk.head
                       : static_cast<T*>(a.dv) + t.b * a.sdv.batch + j_key * a.sdv.token + t.hk * a.sdv.head;
          for (int c = 0; c < a.head_dim; c += 8) {
            if (p.splits > 1) {
              *reinterpret_cast<float4*>(part(c)) = make_float4(0, 0, 0, 0);
              *reinterpret_cast<float4*>(part(c + 4)) = make_float4(0, 0, 0, 0);
            } else {
              *reinterpret_cast<uint4*>(grad + c) = make_uint4(0, 0, 0, 0);
            }
          }
        }
        continue;
      }
      int ds_exp = 0;
      if constexpr (kXScaled<T>) {
        const unsigned int* norm2 = p.max_norm2 + 2 * (static_cast<int64_t>(t.b) * a.kv_heads + t.hk);
        ds_exp = x_ds_exp(__uint_as_float(norm2[0]), __uint_as_float(norm2[1]));
      }
      // from P times its power of two to dS times its own
      const float f_ds = x_exp2i(ds_exp - kXWeightExp);
      for (int j = t.j0; j < t.j1 && ok; ++j, ++g) {
        const int steps = x_row_steps(a, j % p.row_tiles);
        for (int u = 0; u < steps; ++u, ++n) {
          if ((n & 1) != static_cast<uint32_t>(gp)) continue;
          ok = wait(s_full + gp, n >> 1, kWaitS);
          if (!ok) break;
          tc_fence_after();
          const float4* neg_lse =
              reinterpret_cast<const float4*>(stats + g % (Ly::kEntries / 2) * 2 * kXTile + u * 64 + half * 32);
          const float4* neg_delta = neg_lse + kXTile / 4;
          float pr[32];
          {
            uint32_t s[32];
            tmem_read(t_s, s);
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              float4 nl = neg_lse[k >> 2];
              if constexpr (kXScaled<T>)
                nl = make_float4(nl.x + kXWeightExp, nl.y + kXWeightExp, nl.z + kXWeightExp, nl.w + kXWeightExp);
              float x0, x1, x2, x3;
              unpair2(fma2(pair2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), c22, pair2(nl.x, nl.y)), x0, x1);
              unpair2(fma2(pair2(__uint_as_float(s[k + 2]), __uint_as_float(s[k + 3])), c22, pair2(nl.z, nl.w)), x2, x3);
              pr[k] = ex2(x0);
              pr[k + 1] = ex2(x1);
              pr[k + 2] = ex2(x2);
              pr[k + 3] = ex2(x3);
            }
            x_store_operand<T, SPLIT>(t_s, pr);
          }
          ok = wait(dp_full + gp, n >> 1, kWaitDP);
          if (!ok) break;
          tc_fence_after();
          {
            uint32_t dp[32];
            tmem_read(t_dp, dp);
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              const float4 nd = neg_delta[k >> 2];
              unpair2(mul2(pair2(pr[k], pr[k + 1]),
                           add2(pair2(__uint_as_float(dp[k]), __uint_as_float(dp[k + 1])), pair2(nd.x, nd.y))),
                      pr[k], pr[k + 1]);
              unpair2(mul2(pair2(pr[k + 2], pr[k + 3]),
                           add2(pair2(__uint_as_float(dp[k + 2]), __uint_as_float(dp[k + 3])), pair2(nd.z, nd.w))),
                      pr[k + 2], pr[k + 3]);
            }
            if constexpr (kXScaled<T>) {
#pragma unroll
              for (int k = 0; k < 32; ++k) pr[k] *= f_ds;
            }
            x_store_operand<T, SPLIT>(t_dp, pr);
          }
          tmem_st_wait();
          tc_fence_before();
          warp_arrive(ds_full + gp);
        }
      }
      if (!ok) break;
      release_stored();
      ok = wait(acc_full, n_item, kWaitAcc);
      if (!ok) break;
      tc_fence_after();
      const int ks = n_item % Ly::kKVStages;
      const uint4 w = words[n_item % (2 * Ly::kKVStages)];
      const bool kept = ((quad == 0 ? w.x : quad == 1 ? w.y : quad == 2 ? w.z : w.w) >> lane) & 1u;
      // where one key is all there is, its weight is 1 whatever its score
      const bool single = SPLIT && __popc(w.x) + __popc(w.y) + __popc(w.z) + __popc(w.w) == 1;
      // dV goes out from V's tile, dK from K's
      uint8_t* stage = smem + (2 * ks + 1 - gp) * Ly::kTileBytes;
      const float f = !kXScaled<T> ? (gp ? a.scale : 1.0f) : gp ? a.scale * x_exp2i(-ds_exp) : x_exp2i(-kXWeightExp);
      const bool zero = !kept || (gp && single);
#pragma unroll
      for (int c = 0; c < HALVES; ++c) {
        const int col = (half * HALVES + c) * 32;
        uint32_t o[32];
        tmem_read(t_lane + kXDkvV + gp * HALVES * 64 + col, o);
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = zero ? 0u : __float_as_uint(__uint_as_float(o[k]) * f);
        if (p.splits > 1) {
          if (j_key < a.k_len) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              if (col + k < a.head_dim)
                *reinterpret_cast<uint4*>(part(col + k)) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          }
        } else {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) pk[k >> 1] = XType<T>::pack2(__uint_as_float(o[k]), __uint_as_float(o[k + 1]));
          uint8_t* dst = stage + (col >> 6) * 16384;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st_shared_v4(dst + swizzle128_offset(key, ((col & 63) >> 3) + i), pk[4 * i], pk[4 * i + 1], pk[4 * i + 2],
                         pk[4 * i + 3]);
        }
      }
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(staged + gp);
        mbar_arrive(acc_free);
      }
      if (hands_out) {
        ok = mbar_wait(staged + gp, n_item & 1, abort_flag, a.err, kErrXDkv + kWaitStaged);
        if (ok && p.splits == 1) {
          for (int hf = 0; hf < HALVES; ++hf)
            tma_store_4d(gp ? &dk_map : &dv_map, stage + hf * 16384, hf * 64, t.hk, t.tile * kXTile, t.b);
          bulk_commit_group();
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (ok) stored = ks;
      if (Ly::kKVStages == 1) release_stored();
      ++n_item;
    }
    if (hands_out) bulk_wait_group<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kXBwdWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds the splits' partial dV and dK in their order.  One thread per four channels.
template <typename T>
__global__ void __launch_bounds__(256) x_dkv_join_kernel(const XBwdParams p) {
  pdl_sync();
  const XAttnParams& a = p.a;
  const int quads = a.head_dim / 4;
  const int64_t half = static_cast<int64_t>(a.batch) * a.k_len * a.kv_heads * quads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < 2 * half;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const bool is_v = i < half;
    float4 s = make_float4(0, 0, 0, 0);
    for (int k = 0; k < p.splits; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(p.part + 4 * (2 * half * k + i));
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    int64_t r = is_v ? i : i - half;
    const int c = static_cast<int>(r % quads) * 4;
    r /= quads;
    const int hk = static_cast<int>(r % a.kv_heads);
    r /= a.kv_heads;
    const int j = static_cast<int>(r % a.k_len), b = static_cast<int>(r / a.k_len);
    T* dst = is_v ? static_cast<T*>(a.dv) + b * a.sdv.batch + j * a.sdv.token + hk * a.sdv.head
                  : static_cast<T*>(a.dk) + b * a.sdk.batch + j * a.sdk.token + hk * a.sdk.head;
    *reinterpret_cast<uint2*>(dst + c) = make_uint2(XType<T>::pack2(s.x, s.y), XType<T>::pack2(s.z, s.w));
  }
}

}  // namespace fp8b
