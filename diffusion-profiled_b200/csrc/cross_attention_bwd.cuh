// cross_attention_bwd.cuh — gradient of the attention of cross_attention.cuh.
//
// Two launches, each with its sums in tensor memory from beginning to end, so that no
// gradient is added to memory by several CTAs (no atomics, one order of addition):
//   * x_dq_kernel: a row tile of queries against its key tiles.  delta_i = do_i . o_i
//     first (fp32; stored for the second launch with the row's log-sum-exp), then per
//     key tile S = Q K^T and dP = dO V^T, dS = P (dP - delta), dQ += dS K;
//   * x_dkv_kernel: a key tile against the row tiles that read it, all heads that share
//     it among them.  The scores are formed transposed, S^T = K Q^T and dP^T = V dO^T
//     (lane = key), so that P^T and dS^T lie in tensor memory as the first operands of
//     dV += P^T dO and dK += dS^T Q.
// That is seven products a tile pair; a single launch would need five, but would add
// dQ to memory from every key tile.  Both kernels know the rows' log-sum-exp, so no
// maximum is searched and a row of scores needs no single owner: 16 softmax warps take
// 32 columns of a row each (four warps a scheduler hide the exponentials' and loads'
// latency that two with 64 columns do not).  Two
// warps issue the products: one the scores and dP, one the gradients.  In x_dq_kernel the
// scores run ahead into a second buffer; in x_dkv_kernel, where tensor memory has no room
// for one, P^T takes the place of S^T and dS^T that of dP^T, so that dV += P^T dO and the
// next scores run while dS^T is made, and dK += dS^T Q and the next dP^T while the next
// exponentials are.
//
// P and dS are rounded to the tensors' type (they are matrix operands); scores, dP,
// statistics and all sums are fp32.
#pragma once

#include "cross_attention.cuh"

namespace fp8b {

constexpr int kXBwdWarps = 16;                           // softmax warps
constexpr int kXBwdThreads = kXBwdWarps * 32 + 96;       // and loads, scores, gradients

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
};

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

// ============================================================================ dQ
template <int HALVES>
struct XDqLayout {
  static constexpr int kTileBytes = HALVES * 16384;
  static constexpr int kQStages = HALVES == 1 ? 3 : 1;  // Q and dO of an item
  // A key tile stays from its scores to its dQ product, two tiles later; a value tile only for its dP.
  static constexpr int kKStages = HALVES == 1 ? 4 : 3;
  static constexpr int kVStages = HALVES == 1 ? 3 : 2;
  static constexpr int kK = 2 * kQStages * kTileBytes;
  static constexpr int kV = kK + kKStages * kTileBytes;
  static constexpr int kWords = kV + kVStages * kTileBytes;
  static constexpr int kDelta = kWords + kXMaskSlots * 16;  // fp32 [2][128]: the halves of the rows' delta
  static constexpr int kBar = kDelta + 1024;
  static constexpr int kNumBars = 2 * (kQStages + kKStages + kVStages) + 13;
  static constexpr int kTail = kBar + kNumBars * 8;
  static constexpr int kSmemBytes = kTail + 16 + 1024;
};
static_assert(XDqLayout<1>::kSmemBytes <= 232448 && XDqLayout<2>::kSmemBytes <= 232448, "dq smem");
// tensor memory columns: two score buffers (dS over the first half of each 32), dP, dQ
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

template <typename T, int HALVES>
__global__ void __launch_bounds__(kXBwdThreads, 1)
    x_dq_kernel(const XBwdParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap do_map,
                const __grid_constant__ CUtensorMap dq_map) {
  using Ly = XDqLayout<HALVES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint4* words = reinterpret_cast<uint4*>(smem + Ly::kWords);
  float* delta_half = reinterpret_cast<float*>(smem + Ly::kDelta);
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
  uint64_t* ds_full = dp_free + 1;
  uint64_t* acc_full = ds_full + 1;
  uint64_t* acc_free = acc_full + 1;
  uint64_t* staged = acc_free + 1;
  uint64_t* delta_full = staged + 1;
  uint64_t* drained = delta_full + 1;  // [2], by issuing warp
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
      mbar_init(drained + i, 1);
    }
    mbar_init(dp_full, 1);
    mbar_init(dp_free, kXBwdWarps);
    mbar_init(ds_full, kXBwdWarps);
    mbar_init(acc_full, 1);
    mbar_init(acc_free, kXBwdWarps);
    mbar_init(staged, kXBwdWarps);
    mbar_init(delta_full, 8);
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
        if (holes) x_zero_rows<HALVES>(sk, w, x_chunks(t.keys, j) * 32, lane);
        if (g >= 2 && !(ok = wait(s_free + buf, (g >> 1) ^ 1, kWaitSFree))) break;
        tc_fence_after();
        if (elect_one()) {
          products_k_major(tmem + kXDqS + buf * 128, sq, k_major_desc(smem_u32(sk)), idesc, ksteps);
          umma_commit(s_full + buf);
          mbar_arrive(s_full + buf);
        }
        __syncwarp();
        if (!(ok = wait(v_full + vs, g / Ly::kVStages, kWaitV))) break;
        if (holes) x_zero_rows<HALVES>(sv, w, x_chunks(t.keys, j) * 32, lane);
        if (g >= 1 && !(ok = wait(dp_free, g ^ 1, kWaitDPFree))) break;
        tc_fence_after();
        if (elect_one()) {
          products_k_major(tmem + kXDqDP, sdo, k_major_desc(smem_u32(sv)), idesc, ksteps);
          umma_commit(v_empty + vs);
          umma_commit(dp_full);
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
        ok = wait(k_full + ks, g / Ly::kKStages, kWaitK) && wait(ds_full, g, kWaitP);
        if (ok && j == 0 && n_item > 0) ok = wait(acc_free, n_item ^ 1, kWaitAccFree);  // the last item's dQ has been read
        if (!ok) break;
        const uint64_t sk = mn_major_desc(s_base + Ly::kK + ks * Ly::kTileBytes);
        const uint32_t ds = tmem + kXDqS + buf * 128, later = j > 0 ? 1u : 0u;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k)  // dS of 32 columns lies in the first 16 of them
            if (k < steps)
              umma_f16_ts(tmem + kXDqAcc, ds + (k >> 1) * 32 + (k & 1) * 8, sk + k * 128, idesc, k > 0 ? 1u : later);
          umma_commit(s_free + buf);
          umma_commit(k_empty + ks);
          if (j == t.tiles - 1) umma_commit(acc_full);
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
    const auto fetch = [&](const XDqItems& items) {
      XDqItem t;
      const bool exists = items.ahead(t);
      const int token = t.tile * a.tile_tokens + my_token, head = t.hv * a.pack + my_head;
      const bool live = exists && t.tiles > 0 && row < rows && token < a.q_len;
      if (HALVES == 1 && wq < 2) {
        const T* o = static_cast<const T*>(a.o_in) + t.b * a.so.batch + token * a.so.token + head * a.so.head;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = wq * 32 + 8 * u;
          o_row[u] = live && c < a.head_dim ? *reinterpret_cast<const uint4*>(o + c) : make_uint4(0, 0, 0, 0);
        }
      }
      lse = live ? a.lse[(static_cast<int64_t>(t.b) * a.heads + head) * a.q_len + token] : -INFINITY;
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
    bool ok = true;
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
      // ---- delta = do . o, half of the channels each
      if (wq < 2) {
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
        delta_half[wq * kXTile + row] = part;
        __syncwarp();
        if (lane == 0) mbar_arrive(delta_full);
      }
      ok = wait(delta_full, n_item, kWaitDelta);
      if (!ok) break;
      const float neg_delta = dead ? 0.0f : delta_half[row] + delta_half[kXTile + row];
      const float neg_lse = dead ? -INFINITY : -lse * 1.4426950408889634f;
      if (wq == 0) {
        stat[0] = neg_lse;
        stat[kXTile] = neg_delta;
      }
      const uint64_t nl2 = pair2(neg_lse, neg_lse), nd2 = pair2(neg_delta, neg_delta);
      for (int j = 0; j < t.tiles; ++j, ++g) {
        const uint32_t t_s = t_lane + kXDqS + (g & 1) * 128 + wq * 32;
        const bool some = wq < x_chunks(t.keys, j);  // the chunk holds keys
        ok = wait(s_full + (g & 1), g >> 1, kWaitS);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[32];
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
            if (w != ~0u) {
#pragma unroll
              for (int k = 0; k < 32; ++k) s[k] = (w >> k) & 1u ? s[k] : 0u;
            }
          }
        }
        ok = wait(dp_full, g, kWaitDP);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t dp[16];
          if (some) {
            tmem_read(t_lane + kXDqDP + wq * 32 + h * 16, dp);
          }
          if (h == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(dp_free);
          }
          if (some) {
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              const uint64_t d = add2(pair2(__uint_as_float(dp[k]), __uint_as_float(dp[k + 1])), nd2);
              float x0, x1;
              unpair2(mul2(pair2(__uint_as_float(s[16 * h + k]), __uint_as_float(s[16 * h + k + 1])), d), x0, x1);
              s[8 * h + (k >> 1)] = XType<T>::pack2(x0, x1);  // the first 16 become dS
            }
          }
        }
        if (some) {
          tmem_st_32x32b_x16(t_s, reinterpret_cast<const uint32_t(&)[16]>(s));
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_full);
      }
      if (!ok) break;
      fetch(items);
      release_stored();
      ok = wait(acc_full, n_item, kWaitAcc);
      if (!ok) break;
      tc_fence_after();
      // dQ goes out from Q's tile, which every product of the item has read by now: a quarter of the channels each
#pragma unroll
      for (int c = 0; c < HALVES; ++c) {
        const int col = (wq * HALVES + c) * 16;
        uint32_t o[16];
        tmem_read(t_lane + kXDqAcc + col, o);
        uint32_t pk[8];
#pragma unroll
        for (int k = 0; k < 16; k += 2)
          pk[k >> 1] = dead ? 0u : XType<T>::pack2(__uint_as_float(o[k]) * a.scale, __uint_as_float(o[k + 1]) * a.scale);
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
        mbar_arrive(acc_free);
        mbar_arrive(staged);
      }
      if (tid == 0) {
        ok = mbar_wait(staged, n_item & 1, abort_flag, a.err, kErrXDq + kWaitStaged);
        if (ok) {
          for (int hf = 0; hf < HALVES; ++hf)
            tma_store_4d(&dq_map, stage + hf * 16384, hf * 64, t.hv * a.pack, t.tile * a.tile_tokens, t.b);
          bulk_commit_group();
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (ok) stored = qs;
      if (Ly::kQStages == 1) release_stored();
      ++n_item;
    }
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
  static constexpr int kNumBars = 2 * kKVStages + 2 * kEntries + 12;
  static constexpr int kTail = kBar + kNumBars * 8;
  static constexpr int kSmemBytes = kTail + 16 + 1024;
};
static_assert(XDkvLayout<1>::kSmemBytes <= 232448 && XDkvLayout<2>::kSmemBytes <= 232448, "dkv smem");
// tensor memory columns: S^T (P^T over it), dP^T (dS^T over it), dV, dK
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

template <typename T, int HALVES>
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
  uint64_t* s_full = q_empty + Ly::kEntries;
  uint64_t* p_full = s_full + 1;
  uint64_t* p_free = p_full + 1;  // P^T has been multiplied
  uint64_t* dp_full = p_free + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* ds_free = ds_full + 1;  // dS^T has been multiplied
  uint64_t* acc_full = ds_free + 1;
  uint64_t* acc_free = acc_full + 1;
  uint64_t* staged = acc_free + 1;   // [2], by half of the softmax threads
  uint64_t* drained = staged + 2;    // [2], by issuing warp
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
      mbar_init(q_empty + i, 1 + i % 2);  // Q: its dK product (S^T came before); dO: its dP^T and its dV product
    }
    mbar_init(s_full, 2);  // the products' commit, and the issuing thread (keep bits)
    mbar_init(p_full, kXBwdWarps);
    mbar_init(p_free, 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_free, 1);
    mbar_init(ds_full, kXBwdWarps);
    mbar_init(acc_full, 1);
    mbar_init(acc_free, kXBwdWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(staged + i, kXBwdWarps / 2);
      mbar_init(drained + i, 1);
    }
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
    const uint32_t idesc = x_idesc<T>(kXTile, 0, 0);
    uint32_t n_item = 0, g = 0;
    bool ok = true;
    XDkvItems items(p);
    XDkvItem t;
    while (ok && items.next(t)) {
      if (t.j0 >= t.j1) continue;
      const int ks = n_item % Ly::kKVStages;
      ok = wait(kv_full + ks, n_item / Ly::kKVStages, kWaitK);
      if (!ok) break;
      const uint4 w = words[n_item % (2 * Ly::kKVStages)];
      if ((w.x & w.y & w.z & w.w) != 0xffffffffu) {
        // rows past the states were copied as zeros
        x_zero_rows<HALVES>(smem + 2 * ks * Ly::kTileBytes, w, a.k_len - t.tile * kXTile, lane);
        x_zero_rows<HALVES>(smem + (2 * ks + 1) * Ly::kTileBytes, w, a.k_len - t.tile * kXTile, lane);
      }
      const uint64_t sk = k_major_desc(s_base + 2 * ks * Ly::kTileBytes);
      const uint64_t sv = k_major_desc(s_base + (2 * ks + 1) * Ly::kTileBytes);
      for (int j = t.j0; j < t.j1; ++j, ++g) {
        const uint32_t eq = 2 * g % Ly::kEntries, phase = 2 * g / Ly::kEntries;
        ok = wait(q_full + eq, phase, kWaitQ);
        if (ok && g >= 1) ok = wait(p_free, g ^ 1, kWaitSFree);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          products_k_major(tmem + kXDkvS, sk, k_major_desc(s_base + Ly::kQ + eq * Ly::kTileBytes), idesc, ksteps);
          umma_commit(s_full);
          mbar_arrive(s_full);
        }
        __syncwarp();
        ok = wait(q_full + eq + 1, phase, kWaitV);
        if (ok && g >= 1) ok = wait(ds_free, g ^ 1, kWaitDPFree);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          products_k_major(tmem + kXDkvDP, sv, k_major_desc(s_base + Ly::kQ + (eq + 1) * Ly::kTileBytes), idesc, ksteps);
          umma_commit(q_empty + eq + 1);
          umma_commit(dp_full);
        }
        __syncwarp();
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
    uint32_t n_item = 0, g = 0;
    bool ok = true;
    XDkvItems items(p);
    XDkvItem t;
    while (ok && items.next(t)) {
      if (t.j0 >= t.j1) continue;
      for (int j = t.j0; j < t.j1; ++j, ++g) {
        const uint32_t eq = 2 * g % Ly::kEntries, phase = 2 * g / Ly::kEntries;
        const uint64_t sq = mn_major_desc(s_base + Ly::kQ + eq * Ly::kTileBytes);
        const uint64_t sdo = mn_major_desc(s_base + Ly::kQ + (eq + 1) * Ly::kTileBytes);
        const uint32_t later = j > t.j0 ? 1u : 0u;
        // 32 rows' P^T or dS^T lies in the first 16 of their columns
        ok = wait(q_full + eq + 1, phase, kWaitV) && wait(p_full, g, kWaitP);
        if (ok && j == t.j0 && n_item > 0) ok = wait(acc_free, n_item ^ 1, kWaitAccFree);  // the last item's sums have been read
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16_ts(tmem + kXDkvV, tmem + kXDkvS + (k >> 1) * 32 + (k & 1) * 8, sdo + k * 128, idesc, k > 0 ? 1u : later);
          umma_commit(p_free);
          umma_commit(q_empty + eq + 1);
        }
        __syncwarp();
        ok = wait(q_full + eq, phase, kWaitQ) && wait(ds_full, g, kWaitPRest);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16_ts(tmem + kXDkvV + HALVES * 64, tmem + kXDkvDP + (k >> 1) * 32 + (k & 1) * 8, sq + k * 128, idesc,
                        k > 0 ? 1u : later);
          umma_commit(ds_free);
          umma_commit(q_empty + eq);
          if (j == t.j1 - 1) umma_commit(acc_full);
        }
        __syncwarp();
      }
      ++n_item;
    }
    if (!ok && elect_one()) {
      volatile int never = 0;
      umma_commit(drained + 1);
      mbar_wait(drained + 1, 0, &never, a.err, kErrXDkv + kWaitDrain);
    }
  } else {
    // ------------------------------------------------------------ P^T, dS^T: thread = key, the 32 rows of chunk wq
    const int wq = warp >> 2, quad = warp & 3, key = quad * 32 + lane;
    const int is_k = wq >> 1;  // the first half of the threads hands out dV, the second dK
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c2 = a.scale * 1.4426950408889634f;
    const uint64_t c22 = pair2(c2, c2);
    const bool hands_out = (warp & 7) == 0 && lane == 0;
    uint32_t n_item = 0, g = 0;
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
      const int c0 = (wq & 1) * HALVES * 32;  // this thread's channels: [c0, c0 + HALVES * 32)
      const auto part = [&](int c) {          // this key's row of the split's partial sums
        return p.part + ((((static_cast<int64_t>(t.split) * 2 + is_k) * a.batch + t.b) * a.k_len + j_key) * a.kv_heads + t.hk) *
                            a.head_dim + c;
      };
      if (t.j0 >= t.j1) {  // no keys in this tile (or no rows in this split)
        if (j_key < a.k_len) {
          T* grad = is_k ? static_cast<T*>(a.dk) + t.b * a.sdk.batch + j_key * a.sdk.token + t.hk * a.sdk.head
                         : static_cast<T*>(a.dv) + t.b * a.sdv.batch + j_key * a.sdv.token + t.hk * a.sdv.head;
          for (int c = c0; c < min(a.head_dim, c0 + HALVES * 32); c += 8) {
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
      bool kept = false;
      for (int j = t.j0; j < t.j1; ++j, ++g) {
        ok = wait(s_full, g, kWaitS);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_s = t_lane + kXDkvS + wq * 32, t_dp = t_lane + kXDkvDP + wq * 32;
        const float4* neg_lse = reinterpret_cast<const float4*>(stats + g % (Ly::kEntries / 2) * 2 * kXTile + wq * 32);
        const float4* neg_delta = neg_lse + kXTile / 4;
        if (j == t.j0)
          kept = (reinterpret_cast<const uint32_t*>(words + n_item % (2 * Ly::kKVStages))[quad] >> lane) & 1u;
        uint32_t s[32];
        tmem_read(t_s, s);
        uint32_t pk[16];
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 nl = neg_lse[k >> 2];
          float x0, x1, x2, x3;
          unpair2(fma2(pair2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), c22, pair2(nl.x, nl.y)), x0, x1);
          unpair2(fma2(pair2(__uint_as_float(s[k + 2]), __uint_as_float(s[k + 3])), c22, pair2(nl.z, nl.w)), x2, x3);
          x0 = ex2(x0);
          x1 = ex2(x1);
          x2 = ex2(x2);
          x3 = ex2(x3);
          s[k] = __float_as_uint(x0);
          s[k + 1] = __float_as_uint(x1);
          s[k + 2] = __float_as_uint(x2);
          s[k + 3] = __float_as_uint(x3);
          pk[k >> 1] = XType<T>::pack2(x0, x1);
          pk[(k >> 1) + 1] = XType<T>::pack2(x2, x3);
        }
        tmem_st_32x32b_x16(t_s, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
        ok = wait(dp_full, g, kWaitDP);
        if (!ok) break;
        tc_fence_after();
        uint32_t dp[32];
        tmem_read(t_dp, dp);
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 nd = neg_delta[k >> 2];
          float x0, x1, x2, x3;
          unpair2(mul2(pair2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])),
                       add2(pair2(__uint_as_float(dp[k]), __uint_as_float(dp[k + 1])), pair2(nd.x, nd.y))), x0, x1);
          unpair2(mul2(pair2(__uint_as_float(s[k + 2]), __uint_as_float(s[k + 3])),
                       add2(pair2(__uint_as_float(dp[k + 2]), __uint_as_float(dp[k + 3])), pair2(nd.z, nd.w))), x2, x3);
          pk[k >> 1] = XType<T>::pack2(x0, x1);
          pk[(k >> 1) + 1] = XType<T>::pack2(x2, x3);
        }
        tmem_st_32x32b_x16(t_dp, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_full);
      }
      if (!ok) break;
      release_stored();
      ok = wait(acc_full, n_item, kWaitAcc);
      if (!ok) break;
      tc_fence_after();
      const int ks = n_item % Ly::kKVStages;
      // dV goes out from V's tile, dK from K's
      uint8_t* stage = smem + (2 * ks + 1 - is_k) * Ly::kTileBytes;
      const float f = is_k ? a.scale : 1.0f;
#pragma unroll
      for (int c = 0; c < HALVES; ++c) {
        const int col = c0 + c * 32;
        uint32_t o[32];
        tmem_read(t_lane + kXDkvV + is_k * HALVES * 64 + col, o);
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = kept ? __float_as_uint(__uint_as_float(o[k]) * f) : 0u;
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
          uint8_t* half = stage + (col >> 6) * 16384;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            st_shared_v4(half + swizzle128_offset(key, ((col & 63) >> 3) + u), pk[4 * u], pk[4 * u + 1], pk[4 * u + 2],
                         pk[4 * u + 3]);
        }
      }
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(acc_free);
        mbar_arrive(staged + is_k);
      }
      if (hands_out) {
        ok = mbar_wait(staged + is_k, n_item & 1, abort_flag, a.err, kErrXDkv + kWaitStaged);
        if (ok && p.splits == 1) {
          for (int hf = 0; hf < HALVES; ++hf)
            tma_store_4d(is_k ? &dk_map : &dv_map, stage + hf * 16384, hf * 64, t.hk, t.tile * kXTile, t.b);
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
