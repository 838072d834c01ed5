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
// maximum is searched and the 256 softmax threads take 64 columns of a row each.
//
// P and dS are rounded to the tensors' type (they are matrix operands); scores, dP,
// statistics and all sums are fp32.
#pragma once

#include "cross_attention.cuh"

namespace fp8b {

struct XBwdParams {
  XAttnParams a;
  int row_tiles;  // row tiles of a (sequence, head group)
  float2* stats;  // [batch][head groups][row_tiles][128]: (lse in log2 units, +inf where the row has no weight; delta)
  int64_t items;
  // x_dkv_kernel
  int q_tiles;    // row tiles that read a key head: (group / pack) * row_tiles
  int q_chunk;    // row tiles of a split; splits == 1: all of them
  int splits;
  float* part;    // [splits][2][batch][k_len][kv_heads][head_dim] (dv, dk * scale), with splits > 1
};

// Sum of the products of eight 16-bit values.
template <typename T>
__device__ __forceinline__ float x_dot8(const uint4& x, const uint4& y) {
  float s = 0.0f;
  const T* u = reinterpret_cast<const T*>(&x);
  const T* v = reinterpret_cast<const T*>(&y);
#pragma unroll
  for (int k = 0; k < 8; ++k) s = fmaf(to_f32(u[k]), to_f32(v[k]), s);
  return s;
}

// ============================================================================ dQ
template <int HALVES>
struct XDqLayout {
  static constexpr int kTileBytes = HALVES * 16384;
  static constexpr int kQStages = HALVES == 1 ? 3 : 1;  // Q and dO of an item
  static constexpr int kEntries = HALVES == 1 ? 6 : 5;  // key and value tiles in turn
  static constexpr int kKV = 2 * kQStages * kTileBytes;
  static constexpr int kWords = kKV + kEntries * kTileBytes;
  static constexpr int kBar = kWords + kXMaskSlots * 16;
  static constexpr int kNumBars = 2 * kQStages + 2 * kEntries + 9;
  static constexpr int kTail = kBar + kNumBars * 8;
  static constexpr int kSmemBytes = kTail + 16 + 1024;
  static constexpr int kThreads = 320;
};
static_assert(XDqLayout<1>::kSmemBytes <= 232448 && XDqLayout<2>::kSmemBytes <= 232448, "dq smem");
// tensor memory columns: two score buffers (dS over the first half of each 64), dP, dQ
constexpr uint32_t kXDqS = 0, kXDqDP = 256, kXDqAcc = 384;

// A place in the sequence of (item, key tile) pairs of a CTA.
template <typename Item>
struct XCursor {
  int64_t i;
  Item t;
  int j;
  uint32_t g;       // tiles before this one
  uint32_t n_item;  // items with tiles before this one
};
// Moves to the next tile at or after c; false when there is none.
template <typename Item, typename MakeItem>
__device__ __forceinline__ bool x_seek(XCursor<Item>& c, int64_t items, const MakeItem& make) {
  while (c.j >= c.t.j1) {
    c.i += gridDim.x;
    if (c.i >= items) return false;
    if (c.t.j1 > c.t.j0) ++c.n_item;
    c.t = make(c.i);
    c.j = c.t.j0;
  }
  return true;
}

struct XDqItem {
  int b, hv, tile, keys, j0, j1;
};
__device__ __forceinline__ XDqItem x_dq_item(const XBwdParams& p, int64_t i) {
  XDqItem t;
  t.tile = static_cast<int>(i % p.row_tiles);
  i /= p.row_tiles;
  const int hv = p.a.heads / p.a.pack;
  t.hv = static_cast<int>(i % hv);
  t.b = static_cast<int>(i / hv);
  t.keys = x_key_count(p.a, t.b);
  t.j0 = 0;
  t.j1 = (t.keys + kXTile - 1) / kXTile;
  return t;
}

template <typename T, int HALVES>
__global__ void __launch_bounds__(XDqLayout<HALVES>::kThreads, 1)
    x_dq_kernel(const XBwdParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap do_map,
                const __grid_constant__ CUtensorMap dq_map) {
  using Ly = XDqLayout<HALVES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint4* words = reinterpret_cast<uint4*>(smem + Ly::kWords);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + Ly::kBar);
  uint64_t* q_empty = q_full + Ly::kQStages;
  uint64_t* kv_full = q_empty + Ly::kQStages;
  uint64_t* kv_empty = kv_full + Ly::kEntries;
  uint64_t* s_full = kv_empty + Ly::kEntries;  // [2], by score buffer
  uint64_t* dp_full = s_full + 2;
  uint64_t* dp_free = dp_full + 1;
  uint64_t* ds_full = dp_free + 1;
  uint64_t* acc_full = ds_full + 1;
  uint64_t* acc_free = acc_full + 1;
  uint64_t* staged = acc_free + 1;
  uint64_t* drained = staged + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Ly::kTail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < Ly::kQStages; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
    }
    for (int i = 0; i < Ly::kEntries; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
    }
    mbar_init(s_full, 2);
    mbar_init(s_full + 1, 2);
    mbar_init(dp_full, 1);
    mbar_init(dp_free, 8);
    mbar_init(ds_full, 8);
    mbar_init(acc_full, 1);
    mbar_init(acc_free, 8);
    mbar_init(staged, 8);
    mbar_init(drained, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
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
  const auto make = [&](int64_t i) { return x_dq_item(p, i); };

  if (warp == 8) {
    // ------------------------------------------------------------ loads
    const uint32_t q_bytes = static_cast<uint32_t>(a.tile_tokens * a.pack) * 128u * HALVES;
    uint32_t e = 0, loaded = 0, n_item = 0, g = 0;
    bool ok = true;
    for (int64_t i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
      const XDqItem t = make(i);
      if (t.j0 >= t.j1) continue;
      const int qs = n_item % Ly::kQStages;
      ok = warp_wait(q_empty + qs, ((n_item / Ly::kQStages) & 1) ^ 1, abort_flag, a.err, kErrTimeoutProducer);
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
      for (int j = t.j0; j < t.j1 && ok; ++j, ++g) {
        if (masked || (j + 1) * kXTile > t.keys) {
          const uint4 w = x_keep_words(a, t.b, j * kXTile, t.keys, lane);
          if (lane == 0) words[g % kXMaskSlots] = w;
        }
#pragma unroll
        for (int kv = 0; kv < 2 && ok; ++kv, ++e) {
          const int slot = e % Ly::kEntries;
          ok = warp_wait(kv_empty + slot, ((e / Ly::kEntries) & 1) ^ 1, abort_flag, a.err, kErrTimeoutProducer);
          if (!ok) break;
          loaded = e + 1;
          if (lane == 0) {
            mbar_arrive_expect_tx(kv_full + slot, Ly::kTileBytes);
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_4d(smem + Ly::kKV + slot * Ly::kTileBytes + hf * 16384, kv ? &v_map : &k_map, kv_full + slot,
                          hf * 64, hk, j * kXTile, t.b);
          }
        }
      }
    }
    if (!ok && lane == 0) {  // copies still in flight land before the CTA leaves
      volatile int never = 0;
      for (uint32_t k = loaded > Ly::kEntries ? loaded - Ly::kEntries : 0; k < loaded; ++k)
        mbar_wait(kv_full + k % Ly::kEntries, (k / Ly::kEntries) & 1, &never, a.err, kErrTimeoutDrain);
      for (uint32_t k = n_item > Ly::kQStages ? n_item - Ly::kQStages : 0; k < n_item; ++k)
        mbar_wait(q_full + k % Ly::kQStages, (k / Ly::kQStages) & 1, &never, a.err, kErrTimeoutDrain);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ products
    using Cursor = XCursor<XDqItem>;
    const uint32_t s_base = smem_u32(smem);
    bool ok = true;
    uint32_t n_acc = 0;
    const auto wait_entry = [&](uint32_t entry, const Cursor& c) {
      const int slot = entry % Ly::kEntries;
      if (!warp_wait(kv_full + slot, (entry / Ly::kEntries) & 1, abort_flag, a.err, kErrTimeoutMma)) return false;
      if (masked || (c.j + 1) * kXTile > c.t.keys) {
        const uint4 w = words[c.g % kXMaskSlots];
        if ((w.x & w.y & w.z & w.w) != 0xffffffffu) x_zero_rows<HALVES>(smem + Ly::kKV + slot * Ly::kTileBytes, w, lane);
      }
      return true;
    };
    // S of a tile into score buffer g % 2
    const auto issue_s = [&](const Cursor& c) {
      const int qs = c.n_item % Ly::kQStages;
      if (c.j == c.t.j0 && !warp_wait(q_full + qs, (c.n_item / Ly::kQStages) & 1, abort_flag, a.err, kErrTimeoutMma))
        return false;
      if (!wait_entry(2 * c.g, c)) return false;
      if (lane == 0) {
        const uint32_t idesc = x_idesc<T>(x_chunks(c.t.keys, c.j) * 32, 0, 0);
        const uint32_t sq = s_base + 2 * qs * Ly::kTileBytes;
        const uint32_t sk = s_base + Ly::kKV + (2 * c.g % Ly::kEntries) * Ly::kTileBytes;
        tc_fence_after();
        for (int k = 0; k < ksteps; ++k) {
          const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
          umma_f16_ss(tmem + kXDqS + (c.g & 1) * 128, make_smem_desc(sq + off, 16, 1024), make_smem_desc(sk + off, 16, 1024),
                      idesc, k > 0 ? 1u : 0u);
        }
        umma_commit(s_full + (c.g & 1));
        mbar_arrive(s_full + (c.g & 1));
      }
      __syncwarp();
      return true;
    };
    const auto issue_dp = [&](const Cursor& c) {
      if (!wait_entry(2 * c.g + 1, c)) return false;
      if (lane == 0) {
        const uint32_t idesc = x_idesc<T>(x_chunks(c.t.keys, c.j) * 32, 0, 0);
        const uint32_t sdo = s_base + (2 * (c.n_item % Ly::kQStages) + 1) * Ly::kTileBytes;
        const uint32_t entry = 2 * c.g + 1;
        const uint32_t sv = s_base + Ly::kKV + (entry % Ly::kEntries) * Ly::kTileBytes;
        tc_fence_after();
        for (int k = 0; k < ksteps; ++k) {
          const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
          umma_f16_ss(tmem + kXDqDP, make_smem_desc(sdo + off, 16, 1024), make_smem_desc(sv + off, 16, 1024), idesc,
                      k > 0 ? 1u : 0u);
        }
        umma_commit(dp_full);
        umma_commit(kv_empty + entry % Ly::kEntries);
      }
      __syncwarp();
      return true;
    };
    const auto issue_dq = [&](const Cursor& c) {
      if (!warp_wait(ds_full, c.g & 1, abort_flag, a.err, kErrTimeoutMma)) return false;
      if (c.j == c.t.j0) {  // the last item's gradient has been read
        if (n_acc > 0 && !warp_wait(acc_free, (n_acc - 1) & 1, abort_flag, a.err, kErrTimeoutMma)) return false;
        ++n_acc;
      }
      if (lane == 0) {
        const uint32_t idesc = x_idesc<T>(ksteps * 16, 0, 1);
        const uint32_t sk = s_base + Ly::kKV + (2 * c.g % Ly::kEntries) * Ly::kTileBytes;
        const uint32_t ds = tmem + kXDqS + (c.g & 1) * 128;
        tc_fence_after();
        const int steps = 2 * x_chunks(c.t.keys, c.j);
        for (int k = 0; k < steps; ++k)  // dS of columns 64 .. 127 lies at column 64 of the buffer
          umma_f16_ts(tmem + kXDqAcc, ds + (k >> 2) * 64 + (k & 3) * 8, make_smem_desc(sk + k * 2048, 16384, 1024), idesc,
                      (c.j > c.t.j0 || k > 0) ? 1u : 0u);
        umma_commit(kv_empty + 2 * c.g % Ly::kEntries);
        if (c.j == c.t.j1 - 1) umma_commit(acc_full);
      }
      __syncwarp();
      return true;
    };
    const auto next = [&](const Cursor& c, bool* have) {
      Cursor n = c;
      ++n.j;
      ++n.g;
      *have = x_seek(n, p.items, make);
      return n;
    };

    Cursor cur{};
    cur.i = blockIdx.x;
    bool have = cur.i < p.items;
    if (have) {
      cur.t = make(cur.i);
      cur.j = cur.t.j0;
      have = x_seek(cur, p.items, make);
    }
    // With one Q stage, the next item's Q and dO arrive only after this item's gradient has left: its products
    // are issued when the last dQ product of this one has been.
    const auto ahead = [&](const Cursor& from, const Cursor& to) { return Ly::kQStages > 1 || from.i == to.i; };
    if (have) ok = issue_s(cur) && issue_dp(cur);
    bool have1 = false;
    Cursor n1 = cur;
    if (have) n1 = next(cur, &have1);
    bool s1 = false;  // S of the next tile has been issued
    if (ok && have1 && ahead(cur, n1)) {
      ok = issue_s(n1);
      s1 = true;
    }
    while (have && ok) {
      bool have2 = false, dp1 = false;
      Cursor n2 = n1;
      if (have1) n2 = next(n1, &have2);
      if (s1) {
        ok = warp_wait(dp_free, cur.g & 1, abort_flag, a.err, kErrTimeoutMma) && issue_dp(n1);
        dp1 = true;
      }
      ok = ok && issue_dq(cur);
      if (ok && have1 && !s1) ok = issue_s(n1);
      if (ok && have1 && !dp1) ok = issue_dp(n1);  // dS of this tile was waited for: dP is free
      s1 = false;
      if (ok && have2 && ahead(n1, n2)) {
        ok = issue_s(n2);
        s1 = true;
      }
      cur = n1;
      n1 = n2;
      have = have1;
      have1 = have2;
    }
    if (!ok && lane == 0) {  // the products in flight end before the tensor memory is freed
      volatile int never = 0;
      umma_commit(drained);
      mbar_wait(drained, 0, &never, a.err, kErrTimeoutDrain);
    }
  } else {
    // ------------------------------------------------------------ dS: thread = row, 64 columns of half wh
    const int wh = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c2 = a.scale * 1.4426950408889634f;
    const int rows = a.tile_tokens * a.pack;
    const int hv = a.heads / a.pack;
    uint32_t n_item = 0, g = 0;
    bool ok = true;
    for (int64_t i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
      const XDqItem t = make(i);
      const int token = t.tile * a.tile_tokens + row / a.pack, head = t.hv * a.pack + row % a.pack;
      const bool live = row < rows && token < a.q_len;
      float2* stat = p.stats + (((static_cast<int64_t>(t.b) * hv + t.hv) * p.row_tiles + t.tile) * kXTile + row);
      if (t.j0 >= t.j1) {  // no keys
        if (wh == 0) *stat = make_float2(INFINITY, 0.0f);
        if (wh == 0 && live) {
          T* o = static_cast<T*>(a.dq) + t.b * a.sdq.batch + token * a.sdq.token + head * a.sdq.head;
          for (int c = 0; c < a.head_dim; c += 8) *reinterpret_cast<uint4*>(o + c) = make_uint4(0, 0, 0, 0);
        }
        continue;
      }
      float lse2 = INFINITY, delta = 0.0f;
      if (live) {
        const T* o = static_cast<const T*>(a.o_in) + t.b * a.so.batch + token * a.so.token + head * a.so.head;
        const T* d = static_cast<const T*>(a.dout) + t.b * a.sdo.batch + token * a.sdo.token + head * a.sdo.head;
        const float lse = a.lse[(static_cast<int64_t>(t.b) * a.heads + head) * a.q_len + token];
#pragma unroll 8
        for (int c = 0; c < a.head_dim; c += 8)
          delta += x_dot8<T>(__ldg(reinterpret_cast<const uint4*>(o + c)), __ldg(reinterpret_cast<const uint4*>(d + c)));
        if (lse != -INFINITY) lse2 = lse * 1.4426950408889634f;
      }
      if (wh == 0) *stat = make_float2(lse2, delta);
      for (int j = t.j0; j < t.j1; ++j, ++g) {
        const int chunks = x_chunks(t.keys, j);
        const uint32_t t_s = t_lane + kXDqS + (g & 1) * 128 + wh * 64;
        ok = warp_wait(s_full + (g & 1), (g >> 1) & 1, abort_flag, a.err, kErrTimeoutEpilogue);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[2][32], dp[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (2 * wh + c < chunks) tmem_ld_32x32b_x32(t_s + c * 32, s[c]);
        tmem_ld_wait();
        after_wait(s[0]);
        after_wait(s[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k) s[c][k] = __float_as_uint(ex2(fmaf(__uint_as_float(s[c][k]), c2, -lse2)));
        if (masked || (j + 1) * kXTile > t.keys) {
          const uint4 w4 = words[g % kXMaskSlots];
          const uint32_t w[2] = {wh ? w4.z : w4.x, wh ? w4.w : w4.y};
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) s[c][k] = (w[c] >> k) & 1u ? s[c][k] : 0u;
        }
        ok = warp_wait(dp_full, g & 1, abort_flag, a.err, kErrTimeoutEpilogue);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (2 * wh + c < chunks) tmem_ld_32x32b_x32(t_lane + kXDqDP + wh * 64 + c * 32, dp[c]);
        tmem_ld_wait();
        after_wait(dp[0]);
        after_wait(dp[1]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dp_free);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (2 * wh + c < chunks) {
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 32; k += 2)
              pk[k >> 1] = XType<T>::pack2(__uint_as_float(s[c][k]) * (__uint_as_float(dp[c][k]) - delta),
                                           __uint_as_float(s[c][k + 1]) * (__uint_as_float(dp[c][k + 1]) - delta));
            tmem_st_32x32b_x16(t_s + c * 16, pk);
          }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_full);
      }
      if (ok) ok = warp_wait(acc_full, n_item & 1, abort_flag, a.err, kErrTimeoutEpilogue);
      if (!ok) break;
      tc_fence_after();
      const int qs = n_item % Ly::kQStages;
      uint8_t* stage = smem + 2 * qs * Ly::kTileBytes;  // Q's tile, read by every product of the item by now
#pragma unroll
      for (int c = 0; c < HALVES; ++c) {  // this half's share of the channels: [wh * HALVES * 32, + HALVES * 32)
        const int col = (wh * HALVES + c) * 32;
        uint32_t o[32];
        tmem_ld_32x32b_x32(t_lane + kXDqAcc + col, o);
        tmem_ld_wait();
        after_wait(o);
        uint32_t pk[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2)
          pk[k >> 1] = lse2 == INFINITY ? 0u : XType<T>::pack2(__uint_as_float(o[k]) * a.scale, __uint_as_float(o[k + 1]) * a.scale);
        uint8_t* half = stage + (col >> 6) * 16384;
#pragma unroll
        for (int u = 0; u < 4; ++u)
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
        ok = mbar_wait(staged, n_item & 1, abort_flag, a.err, kErrTimeoutEpilogue);
        if (ok) {
          for (int hf = 0; hf < HALVES; ++hf)
            tma_store_4d(&dq_map, stage + hf * 16384, hf * 64, t.hv * a.pack, t.tile * a.tile_tokens, t.b);
          bulk_commit_group();
          bulk_wait_group_read<0>();
          mbar_arrive(q_empty + qs);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      ++n_item;
    }
    if (tid == 0) bulk_wait_group<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
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
  static constexpr int kStats = kQ + kEntries * kTileBytes;  // float2 [kEntries / 2][128]
  static constexpr int kWords = kStats + kEntries / 2 * 1024;
  static constexpr int kBar = kWords + 2 * kKVStages * 16;
  static constexpr int kNumBars = 2 * kKVStages + 2 * kEntries + 8;
  static constexpr int kTail = kBar + kNumBars * 8;
  static constexpr int kSmemBytes = kTail + 16 + 1024;
  static constexpr int kThreads = 320;
};
static_assert(XDkvLayout<1>::kSmemBytes <= 232448 && XDkvLayout<2>::kSmemBytes <= 232448, "dkv smem");
// tensor memory columns: S^T, dP^T (P^T and dS^T over it), dV, dK
constexpr uint32_t kXDkvS = 0, kXDkvDP = 128, kXDkvV = 256;

struct XDkvItem {
  int b, hk, tile, split, keys, j0, j1;  // row tiles [j0, j1) of the key head; none where the tile has no keys
};
__device__ __forceinline__ XDkvItem x_dkv_item(const XBwdParams& p, int64_t i) {
  XDkvItem t;
  const int tiles = (p.a.k_len + kXTile - 1) / kXTile;
  t.tile = static_cast<int>(i % tiles);
  i /= tiles;
  t.split = static_cast<int>(i % p.splits);
  i /= p.splits;
  t.hk = static_cast<int>(i % p.a.kv_heads);
  t.b = static_cast<int>(i / p.a.kv_heads);
  t.keys = x_key_count(p.a, t.b);
  t.j0 = min(p.q_tiles, t.split * p.q_chunk);
  t.j1 = t.tile * kXTile < t.keys ? min(p.q_tiles, t.j0 + p.q_chunk) : t.j0;
  return t;
}

template <typename T, int HALVES>
__global__ void __launch_bounds__(XDkvLayout<HALVES>::kThreads, 1)
    x_dkv_kernel(const XBwdParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap do_map,
                 const __grid_constant__ CUtensorMap dk_map, const __grid_constant__ CUtensorMap dv_map) {
  using Ly = XDkvLayout<HALVES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float2* stats = reinterpret_cast<float2*>(smem + Ly::kStats);
  uint4* words = reinterpret_cast<uint4*>(smem + Ly::kWords);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + Ly::kBar);
  uint64_t* kv_empty = kv_full + Ly::kKVStages;
  uint64_t* q_full = kv_empty + Ly::kKVStages;
  uint64_t* q_empty = q_full + Ly::kEntries;
  uint64_t* s_full = q_empty + Ly::kEntries;
  uint64_t* s_free = s_full + 1;
  uint64_t* dp_full = s_free + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* acc_full = ds_full + 1;
  uint64_t* acc_free = acc_full + 1;
  uint64_t* staged = acc_free + 1;
  uint64_t* drained = staged + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Ly::kTail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const XAttnParams& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = a.tile_tokens * a.pack;
  if (tid == 0) {
    for (int i = 0; i < Ly::kKVStages; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 2);
    }
    for (int i = 0; i < Ly::kEntries; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
    }
    mbar_init(s_full, 2);
    mbar_init(s_free, 8);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 8);
    mbar_init(acc_full, 1);
    mbar_init(acc_free, 8);
    mbar_init(staged, 8);
    mbar_init(drained, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  // rows that no copy fills (128 is not a multiple of `pack`) are zero: they are summed over
  for (int c = tid; c < (kXTile - rows) * 8 * HALVES * Ly::kEntries; c += Ly::kThreads) {
    const int r = rows + c / 8 % (kXTile - rows), tile = c / 8 / (kXTile - rows);
    *reinterpret_cast<uint4*>(smem + Ly::kQ + tile * 16384 + r * 128 + c % 8 * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  const int ksteps = (a.head_dim + 15) >> 4;
  const auto make = [&](int64_t i) { return x_dkv_item(p, i); };

  if (warp == 8) {
    // ------------------------------------------------------------ loads
    const uint32_t q_bytes = static_cast<uint32_t>(rows) * 128u * HALVES;
    const int per_key_head = a.group / a.pack;  // head groups that read a key head (1 where all are packed)
    const int hv = a.heads / a.pack;
    uint32_t e = 0, loaded = 0, n_item = 0;
    bool ok = true;
    for (int64_t i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
      const XDkvItem t = make(i);
      if (t.j0 >= t.j1) continue;
      const int ks = n_item % Ly::kKVStages;
      const uint4 w = x_keep_words(a, t.b, t.tile * kXTile, t.keys, lane);
      ok = warp_wait(kv_empty + ks, ((n_item / Ly::kKVStages) & 1) ^ 1, abort_flag, a.err, kErrTimeoutProducer);
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
        for (int which = 0; which < 2 && ok; ++which, ++e) {
          const int slot = e % Ly::kEntries;
          ok = warp_wait(q_empty + slot, ((e / Ly::kEntries) & 1) ^ 1, abort_flag, a.err, kErrTimeoutProducer);
          if (!ok) break;
          loaded = e + 1;
          if (lane == 0) {
            mbar_arrive_expect_tx(q_full + slot, q_bytes + (which == 0 ? 1024u : 0u));
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_4d(smem + Ly::kQ + slot * Ly::kTileBytes + hf * 16384, which ? &do_map : &q_map, q_full + slot,
                          hf * 64, h * a.pack, tile * a.tile_tokens, t.b);
            if (which == 0)
              bulk_load_1d(stats + (slot >> 1) * kXTile,
                           p.stats + ((static_cast<int64_t>(t.b) * hv + h) * p.row_tiles + tile) * kXTile, 1024,
                           q_full + slot);
          }
        }
      }
    }
    if (!ok && lane == 0) {  // copies still in flight land before the CTA leaves
      volatile int never = 0;
      for (uint32_t k = loaded > Ly::kEntries ? loaded - Ly::kEntries : 0; k < loaded; ++k)
        mbar_wait(q_full + k % Ly::kEntries, (k / Ly::kEntries) & 1, &never, a.err, kErrTimeoutDrain);
      for (uint32_t k = n_item > Ly::kKVStages ? n_item - Ly::kKVStages : 0; k < n_item; ++k)
        mbar_wait(kv_full + k % Ly::kKVStages, (k / Ly::kKVStages) & 1, &never, a.err, kErrTimeoutDrain);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ products
    using Cursor = XCursor<XDkvItem>;
    const uint32_t s_base = smem_u32(smem);
    const uint32_t idesc_s = x_idesc<T>(kXTile, 0, 0), idesc_acc = x_idesc<T>(ksteps * 16, 0, 1);
    bool ok = true;
    uint32_t n_acc = 0;
    const auto wait_entry = [&](uint32_t entry) {
      return warp_wait(q_full + entry % Ly::kEntries, (entry / Ly::kEntries) & 1, abort_flag, a.err, kErrTimeoutMma);
    };
    // D[128 keys][128 rows] = (K or V) (Q or dO)^T
    const auto product_t = [&](uint32_t d, uint32_t sa, uint32_t sb) {
      for (int k = 0; k < ksteps; ++k) {
        const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
        umma_f16_ss(tmem + d, make_smem_desc(sa + off, 16, 1024), make_smem_desc(sb + off, 16, 1024), idesc_s,
                    k > 0 ? 1u : 0u);
      }
    };
    const auto issue_s = [&](const Cursor& c) {
      const int ks = c.n_item % Ly::kKVStages;
      if (c.j == c.t.j0) {
        if (!warp_wait(kv_full + ks, (c.n_item / Ly::kKVStages) & 1, abort_flag, a.err, kErrTimeoutMma)) return false;
        const uint4 w = words[c.n_item % (2 * Ly::kKVStages)];
        if ((w.x & w.y & w.z & w.w) != 0xffffffffu) {
          x_zero_rows<HALVES>(smem + 2 * ks * Ly::kTileBytes, w, lane);
          x_zero_rows<HALVES>(smem + (2 * ks + 1) * Ly::kTileBytes, w, lane);
        }
      }
      if (!wait_entry(2 * c.g)) return false;
      if (lane == 0) {
        tc_fence_after();
        product_t(kXDkvS, s_base + 2 * ks * Ly::kTileBytes, s_base + Ly::kQ + (2 * c.g % Ly::kEntries) * Ly::kTileBytes);
        umma_commit(s_full);
        mbar_arrive(s_full);
      }
      __syncwarp();
      return true;
    };
    const auto issue_dp = [&](const Cursor& c) {
      if (!wait_entry(2 * c.g + 1)) return false;
      if (lane == 0) {
        tc_fence_after();
        product_t(kXDkvDP, s_base + (2 * (c.n_item % Ly::kKVStages) + 1) * Ly::kTileBytes,
                  s_base + Ly::kQ + ((2 * c.g + 1) % Ly::kEntries) * Ly::kTileBytes);
        umma_commit(dp_full);
      }
      __syncwarp();
      return true;
    };
    const auto issue_acc = [&](const Cursor& c) {
      if (!warp_wait(ds_full, c.g & 1, abort_flag, a.err, kErrTimeoutMma)) return false;
      if (c.j == c.t.j0) {  // the last item's gradients have been read
        if (n_acc > 0 && !warp_wait(acc_free, (n_acc - 1) & 1, abort_flag, a.err, kErrTimeoutMma)) return false;
        ++n_acc;
      }
      if (lane == 0) {
        const uint32_t sq = s_base + Ly::kQ + (2 * c.g % Ly::kEntries) * Ly::kTileBytes;
        const uint32_t sdo = s_base + Ly::kQ + ((2 * c.g + 1) % Ly::kEntries) * Ly::kTileBytes;
        const uint32_t acc = c.j > c.t.j0 ? 1u : 0u;
        tc_fence_after();
        // rows 64 h .. 64 h + 63: P^T at column 64 h of the dP region, dS^T at 64 h + 32
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_f16_ts(tmem + kXDkvV, tmem + kXDkvDP + (k >> 2) * 64 + (k & 3) * 8, make_smem_desc(sdo + k * 2048, 16384, 1024),
                      idesc_acc, acc | (k > 0 ? 1u : 0u));
        umma_commit(q_empty + (2 * c.g + 1) % Ly::kEntries);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_f16_ts(tmem + kXDkvV + HALVES * 64, tmem + kXDkvDP + 32 + (k >> 2) * 64 + (k & 3) * 8,
                      make_smem_desc(sq + k * 2048, 16384, 1024), idesc_acc, acc | (k > 0 ? 1u : 0u));
        umma_commit(q_empty + 2 * c.g % Ly::kEntries);
        if (c.j == c.t.j1 - 1) umma_commit(acc_full);
      }
      __syncwarp();
      return true;
    };

    Cursor cur{};
    cur.i = blockIdx.x;
    bool have = cur.i < p.items;
    if (have) {
      cur.t = make(cur.i);
      cur.j = cur.t.j0;
      have = x_seek(cur, p.items, make);
    }
    if (have) ok = issue_s(cur);
    while (have && ok) {
      ok = issue_dp(cur);
      Cursor nxt = cur;
      ++nxt.j;
      ++nxt.g;
      const bool more = x_seek(nxt, p.items, make);
      // with one K / V stage the next item's tiles arrive only after this item's gradients have left
      const bool apart = Ly::kKVStages == 1 && more && nxt.j == nxt.t.j0;
      const auto next_s = [&]() {
        return warp_wait(s_free, cur.g & 1, abort_flag, a.err, kErrTimeoutMma) && issue_s(nxt);
      };
      if (ok && more && !apart) ok = next_s();
      ok = ok && issue_acc(cur);
      if (ok && more && apart) ok = next_s();
      cur = nxt;
      have = more;
    }
    if (!ok && lane == 0) {  // the products in flight end before the tensor memory is freed
      volatile int never = 0;
      umma_commit(drained);
      mbar_wait(drained, 0, &never, a.err, kErrTimeoutDrain);
    }
  } else {
    // ------------------------------------------------------------ P^T, dS^T: thread = key, 64 rows of half wh
    const int wh = warp >> 2, quad = warp & 3, key = quad * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c2 = a.scale * 1.4426950408889634f;
    uint32_t n_item = 0, g = 0;
    bool ok = true;
    for (int64_t i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
      const XDkvItem t = make(i);
      const int j_key = t.tile * kXTile + key;
      T* const grad = wh == 0 ? static_cast<T*>(a.dv) + t.b * a.sdv.batch + static_cast<int64_t>(j_key) * a.sdv.token + t.hk * a.sdv.head
                              : static_cast<T*>(a.dk) + t.b * a.sdk.batch + static_cast<int64_t>(j_key) * a.sdk.token + t.hk * a.sdk.head;
      const auto part = [&](int c) {  // this row of the split's partial sums
        return p.part + ((((static_cast<int64_t>(t.split) * 2 + wh) * a.batch + t.b) * a.k_len + j_key) * a.kv_heads + t.hk) *
                            a.head_dim + c;
      };
      if (t.j0 >= t.j1) {  // no keys in this tile (or no rows in this split)
        if (j_key < a.k_len) {
          if (p.splits > 1) {
            for (int c = 0; c < a.head_dim; c += 4) *reinterpret_cast<float4*>(part(c)) = make_float4(0, 0, 0, 0);
          } else {
            for (int c = 0; c < a.head_dim; c += 8) *reinterpret_cast<uint4*>(grad + c) = make_uint4(0, 0, 0, 0);
          }
        }
        continue;
      }
      bool kept = false;
      for (int j = t.j0; j < t.j1; ++j, ++g) {
        ok = warp_wait(s_full, g & 1, abort_flag, a.err, kErrTimeoutEpilogue);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[2][32], dp[2][32];
        tmem_ld_32x32b_x32(t_lane + kXDkvS + wh * 64, s[0]);
        tmem_ld_32x32b_x32(t_lane + kXDkvS + wh * 64 + 32, s[1]);
        tmem_ld_wait();
        after_wait(s[0]);
        after_wait(s[1]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        if (j == t.j0) {
          const uint4 w = words[n_item % (2 * Ly::kKVStages)];
          kept = ((quad == 0 ? w.x : quad == 1 ? w.y : quad == 2 ? w.z : w.w) >> lane) & 1u;
        }
        const float4* st = reinterpret_cast<const float4*>(stats + (g % (Ly::kEntries / 2)) * kXTile + wh * 64);
        uint32_t pk[2][16];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float4 r = st[c * 16 + (k >> 1)];  // (lse, delta) of two rows
            const float p0 = ex2(fmaf(__uint_as_float(s[c][k]), c2, -r.x));
            const float p1 = ex2(fmaf(__uint_as_float(s[c][k + 1]), c2, -r.z));
            s[c][k] = __float_as_uint(p0);
            s[c][k + 1] = __float_as_uint(p1);
            pk[c][k >> 1] = XType<T>::pack2(p0, p1);
          }
        ok = warp_wait(dp_full, g & 1, abort_flag, a.err, kErrTimeoutEpilogue);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_dp = t_lane + kXDkvDP + wh * 64;
        tmem_ld_32x32b_x32(t_dp, dp[0]);
        tmem_ld_32x32b_x32(t_dp + 32, dp[1]);
        tmem_ld_wait();
        after_wait(dp[0]);
        after_wait(dp[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tmem_st_32x32b_x16(t_dp + c * 16, pk[c]);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float4 r = st[c * 16 + (k >> 1)];
            pk[c][k >> 1] = XType<T>::pack2(__uint_as_float(s[c][k]) * (__uint_as_float(dp[c][k]) - r.y),
                                            __uint_as_float(s[c][k + 1]) * (__uint_as_float(dp[c][k + 1]) - r.w));
          }
          tmem_st_32x32b_x16(t_dp + 32 + c * 16, pk[c]);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_full);
      }
      if (ok) ok = warp_wait(acc_full, n_item & 1, abort_flag, a.err, kErrTimeoutEpilogue);
      if (!ok) break;
      tc_fence_after();
      const int ks = n_item % Ly::kKVStages;
      // dV goes out by the first half of the threads from V's tile, dK by the second from K's
      uint8_t* stage = smem + (2 * ks + 1 - wh) * Ly::kTileBytes;
      const float f = !kept ? 0.0f : wh == 0 ? 1.0f : a.scale;
#pragma unroll
      for (int c = 0; c < 2 * HALVES; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(t_lane + kXDkvV + wh * HALVES * 64 + c * 32, o);
        tmem_ld_wait();
        after_wait(o);
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = kept ? __float_as_uint(__uint_as_float(o[k]) * f) : 0u;
        if (p.splits > 1) {
          if (j_key < a.k_len)
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              if (c * 32 + k < a.head_dim)
                *reinterpret_cast<uint4*>(part(c * 32 + k)) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        } else {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) pk[k >> 1] = XType<T>::pack2(__uint_as_float(o[k]), __uint_as_float(o[k + 1]));
          uint8_t* half = stage + (c >> 1) * 16384;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            st_shared_v4(half + swizzle128_offset(key, (c & 1) * 4 + u), pk[4 * u], pk[4 * u + 1], pk[4 * u + 2],
                         pk[4 * u + 3]);
        }
      }
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(acc_free);
        mbar_arrive(staged);
      }
      if (quad == 0 && lane == 0) {
        ok = mbar_wait(staged, n_item & 1, abort_flag, a.err, kErrTimeoutEpilogue);
        if (ok) {
          if (p.splits == 1) {
            for (int hf = 0; hf < HALVES; ++hf)
              tma_store_4d(wh == 0 ? &dv_map : &dk_map, stage + hf * 16384, hf * 64, t.hk, t.tile * kXTile, t.b);
            bulk_commit_group();
            bulk_wait_group_read<0>();
          }
          mbar_arrive(kv_empty + ks);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      ++n_item;
    }
    if (quad == 0 && lane == 0) bulk_wait_group<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
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
