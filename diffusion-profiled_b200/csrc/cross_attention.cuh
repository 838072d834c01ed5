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
//
// Rows.  The `pack` query heads that share a key head are rows of one tile: row
// r = token * pack + head-in-group, floor(128 / pack) tokens a tile, so that keys and
// values are read once for all of them and their gradients need no second sum.
//
// Forward (x_fwd_kernel): one pass over the keys with a running maximum and sum.
//   * S = Q K^T of 128 rows and 64 keys on tcgen05 kind::f16 into TMEM (fp32); one thread
//     owns one row, reads its 64 scores, and writes P (rounded to the tensors' type, the
//     tensor cores' operand) over them, where the second product O += P V takes it from;
//   * two score buffers: the products of the next 64 keys run while the softmax of these
//     does.  (With one buffer of 128 keys the softmax, P V and the next S are one chain:
//     170 us against 154 for 2 x 4096 queries of 8 heads of 128 over 4096 keys.)  64 keys
//     cost S a third of its rate (its operands' shared-memory reads), which the overlap
//     more than returns;
//   * the exponent's reference is the row's maximum so far, raised only when a score
//     passes it by more than 2^8: then O and the sum are rescaled.  Scores that stay
//     within that factor need no rescaling pass.  P <= 2^8 keeps its relative precision
//     in bf16; in fp16 what is below 2^-14 is a multiple of 2^-24, beside a sum of 1 or more;
//   * keys that are not kept: their scores are replaced by -inf, and their rows of V are
//     zeroed in shared memory before the product.
// What bounds it: with many queries the softmax (an exponential a score, 16 a clock and
// SM) and the products by turns: the 2 x 4096 x 4096 above takes 135 us in a loop of its own,
// 1,018 TFLOP/s, 61 % of the measured peak, and 150 among the gradient's launches; 13 % of it
// is the last wave (512 row tiles on 296 CTAs);
// with few keys the beginning and end of an item (3,000 of 8,000 cycles at 160 keys), which
// the other CTA of the SM fills in part; with single queries the bytes of K and V and the
// latency of a step (32 queries of 16 heads over 8192 keys of 4: 342 MB in 96 us, 3.6 TB/s,
// and 5 us for the join).
// The sums and statistics are fp32; P is the one value rounded before a sum (it is a
// matrix operand).  Over many keys that rounding averages out against the output's own.
// Where the states are at most one key tile it would not, and the products are cheap; with
// few rows a sequence the tensor cores idle.  There (SPLIT) P goes in as the sum of two
// values of the type, P V = P_hi V + P_lo V: the output's error is that of its own rounding
// (1.7e-3 of its norm in bf16, 2.3e-3 with P rounded once), for 8 % of the time of the 32
// queries above (92 us before), none of one query's over 1,024 keys.  For whole tiles of
// rows over several key tiles two values would cost 15 to 24 % (64 x 1024 queries over 256
// keys 41.6 -> 48.0 us, 2 x 4096 x 4096 135 -> 167): there P is rounded once.
//
// Every mbarrier wait is bounded (mbar_wait); on a timeout the kernel records the error
// code, skips the remaining work and frees its tensor memory.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "dropout.cuh"
#include "sm100_common.cuh"

namespace fp8b {

constexpr int kXTile = 128;  // rows of a query tile and keys of a key tile

// Device error codes of the bounded waits: kernel base + the barrier that was waited for.
enum XError : int { kErrXForward = 300, kErrXDq = 320, kErrXDkv = 340 };
enum XWait : int {
  kWaitQFree = 1, kWaitKFree, kWaitVFree, kWaitQ, kWaitK, kWaitV, kWaitS, kWaitSFree, kWaitDP, kWaitDPFree, kWaitP,
  kWaitPV, kWaitAcc, kWaitAccFree, kWaitStaged, kWaitDelta, kWaitDrain
};

struct XStrides {
  int64_t batch, token, head;  // elements
};

struct XAttnParams {
  const void *q, *k, *v, *o_in, *dout;
  void *o, *dq, *dk, *dv;
  XStrides sq, sk, sv, so, sdo, sdq, sdk, sdv;
  float* lse;  // [batch][heads][q_len]
  const int32_t* key_lengths;
  const uint8_t* key_mask;
  int64_t mask_stride;
  int batch, q_len, k_len, heads, kv_heads, head_dim;
  int group;       // query heads per key head
  int pack;        // query heads side by side in a row tile (group, or 1 where group > 128)
  int tile_tokens; // tokens of a row tile: 128 / pack
  float scale;
  int* err;
};

// A sequence's key count as given, and clamped.  (Apart, so that the load can be under way before it is needed.)
__device__ __forceinline__ int x_raw_count(const XAttnParams& p, int b) {
  return p.key_lengths == nullptr ? p.k_len : __ldg(p.key_lengths + b);
}
__device__ __forceinline__ int x_key_count(const XAttnParams& p, int raw) { return max(0, min(p.k_len, raw)); }
__device__ __forceinline__ bool x_key_kept(const XAttnParams& p, int b, int j) {
  return p.key_mask == nullptr || p.key_mask[b * p.mask_stride + j] != 0;
}

// ---------------------------------------------------------------- tcgen05, 16-bit operands
template <typename T>
struct XType;
template <>
struct XType<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1u;
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <>
struct XType<__half> {
  static constexpr uint32_t kFormat = 0u;
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Two fp32 values as the sum of two pairs of T: hi = RN(x), lo = RN(x - hi).
template <typename T>
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = XType<T>::pack2(x0, x1);
  const T* h = reinterpret_cast<const T*>(&hi);
  lo = XType<T>::pack2(x0 - to_f32(h[0]), x1 - to_f32(h[1]));
}

// kind::f16 instruction descriptor for operands of type T, f32 accumulator, M = 128.
template <typename T>
__device__ __forceinline__ uint32_t x_idesc(int n, int a_mn_major, int b_mn_major) {
  return (1u << 4) | (XType<T>::kFormat << 7) | (XType<T>::kFormat << 10) |
         (static_cast<uint32_t>(a_mn_major) << 15) | (static_cast<uint32_t>(b_mn_major) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kXTile >> 4) << 24);
}

// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void umma_f16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]: A's 16-bit elements lie two to a column, row r in lane r
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The warp index as a value the compiler knows to be the same in the whole warp, so that a role's branch and what
// its loops count stay in uniform registers, where the operands of tcgen05.mma have to be.
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0); }

// True in one lane of a converged warp, the same lane every time.  (With `lane == 0` in its place the operands of
// every product are moved to uniform registers one by one: 120 cycles a product of 64 cycles.)
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}

// Descriptor of a 128-byte-swizzled operand tile of [128 rows][64 channels] halves 16 KB apart; read along its rows
// (K-major: 16-channel steps) or across them (MN-major: 16-row steps).
__device__ __forceinline__ uint64_t k_major_desc(uint32_t saddr) { return make_smem_desc(saddr, 16, 1024); }
__device__ __forceinline__ uint64_t mn_major_desc(uint32_t saddr) { return make_smem_desc(saddr, 16384, 1024); }

// D[128][n] = A B^T over `steps` 16-channel steps of two K-major tiles (one elected thread).
__device__ __forceinline__ void products_k_major(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, int steps) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
    if (k < steps) umma_f16_ss(d_tmem, a + off, b + off, idesc, k > 0 ? 1u : 0u);
  }
}

// 32 lanes x 32 (16) columns, TMEM -> register, and the wait for them.  One statement, so that nothing can use the
// registers before the wait.
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// 32 lanes x 16 columns, register -> TMEM.
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Tiled TMA store of a {channels, heads, tokens, batch} box.
__device__ __forceinline__ void tma_store_4d(const void* tmap, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two fp32 values in one 64-bit register, for the packed fp32 instructions.
__device__ __forceinline__ uint64_t pair2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair2(uint64_t p, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// A wait whose outcome the whole warp shares (the loads of tensor memory are warp-wide).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err,
                                          int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code));
}

// A number written in mixed radix, (d0, d1, d2, d3) with radices r0, r1, r2: an item's place (row tile, split, head,
// sequence).  A CTA goes from item to item by adding the grid's digits, without a division.
struct XCount {
  int d0, d1, d2, d3;
};
__device__ __forceinline__ XCount x_count(uint32_t i, uint32_t r0, uint32_t r1, uint32_t r2) {
  XCount c;
  c.d0 = static_cast<int>(i % r0);
  i /= r0;
  c.d1 = static_cast<int>(i % r1);
  i /= r1;
  c.d2 = static_cast<int>(i % r2);
  c.d3 = static_cast<int>(i / r2);
  return c;
}
__device__ __forceinline__ void x_advance(XCount& c, const XCount& by, int r0, int r1, int r2) {
  c.d0 += by.d0;
  const int a = c.d0 >= r0;
  c.d0 -= a ? r0 : 0;
  c.d1 += by.d1 + a;
  const int b = c.d1 >= r1;
  c.d1 -= b ? r1 : 0;
  c.d2 += by.d2 + b;
  const int e = c.d2 >= r2;
  c.d2 -= e ? r2 : 0;
  c.d3 += by.d3 + e;
}

// The 128 keep bits of the keys [j0, j0 + 128) of sequence b (whole warp).
__device__ __forceinline__ uint4 x_keep_words(const XAttnParams& p, int b, int j0, int count, int lane) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = j0 + 32 * i + lane;
    w[i] = __ballot_sync(0xffffffffu, j < count && x_key_kept(p, b, j));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Zeroes the rows below `used` of a [128][64 * HALVES] tile (128-byte rows, halves 16 KB apart) whose keep bit is 0
// (whole warp): a weight of zero times an infinity or NaN stored there would not be zero.  Four rows a step, eight
// lanes a row: a row's 128 bytes meet all banks once.  (One row a lane took 2,000 cycles for 51 rows, this takes 150.)
template <int HALVES>
__device__ __forceinline__ void x_zero_rows(uint8_t* tile, const uint4& keep, int used, int lane) {
  const uint32_t w[4] = {keep.x, keep.y, keep.z, keep.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (32 * i >= used || w[i] == 0xffffffffu) continue;
#pragma unroll
    for (int r = 0; r < 32; r += 4) {
      if (((w[i] >> r) & 15u) == 15u) continue;
      if (!((w[i] >> (r + (lane >> 3))) & 1u))
#pragma unroll
        for (int hf = 0; hf < HALVES; ++hf)
          st_shared_v4(tile + hf * 16384 + (32 * i + r) * 128 + lane * 16, 0, 0, 0, 0);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// ============================================================================ forward
constexpr int kXMaskSlots = 8;  // key tiles whose keep bits are held: more than are ever between load and use

struct XFwdParams {
  XAttnParams a;
  int row_tiles;    // row tiles of a (sequence, head group)
  int hv;           // head groups: heads / pack
  int key_chunk;    // key tiles of a split; splits == 1: all of them
  int splits;
  float* part_o;    // [splits][batch * heads * q_len][head_dim], with splits > 1
  float* part_lse;  // [splits][batch * heads * q_len], base-2 logarithm
  int64_t rows;     // batch * heads * q_len
  uint32_t items;   // (sequence, head group, row tile group, split)
  int join;         // the launch itself joins the splits, which are the CTAs of a cluster (x_join)
};
constexpr int kXMaxSplits = 128;  // four a lane

// A CTA works on one row tile of HALVES * 64 channels at a time, and an SM holds two CTAs: while one begins or ends an
// item, the other computes.  (One CTA with two row tiles, which share its key and value tiles, took 3 to 16 % longer:
// their items begin and end together.  64 x 1024 queries of 4 heads of 64 over up to 256 keys: 39.6 us against 38.2;
// of 128 over 77 keys: 57 against 50.)
template <int HALVES>
struct XFwdLayout {
  static constexpr int kTileBytes = HALVES * 16384;
  static constexpr int kQStages = HALVES == 2 ? 1 : 2;
  static constexpr int kEntries = HALVES == 1 ? 4 : 2;  // key / value tiles: as many as fit half of the SM
  static constexpr int kWarps = 4;                      // softmax warps
  static constexpr int kKV = kTileBytes * kQStages;
  static constexpr int kWords = kKV + kEntries * kTileBytes;
  static constexpr int kBar = kWords + kXMaskSlots * 16;
  static constexpr int kNumBars = 2 * kQStages + 2 * kEntries + 10;
  static constexpr int kTail = kBar + kNumBars * 8;
  static constexpr int kSmemBytes = kTail + 16 + 1024;  // + alignment slack
  static constexpr int kThreads = kWarps * 32 + 64;     // softmax, loads, products
  static constexpr uint32_t kTmemCols = 256;            // two score buffers of 64, output
};
constexpr int kXFwdCtasPerSm = 2;
static_assert(XFwdLayout<2>::kSmemBytes <= 115712 && XFwdLayout<1>::kSmemBytes <= 115712, "two CTAs per SM");

// One unit of work: a row tile of a head group against the key tiles [j0, j1).
struct XItem {
  int b, hv, tile, split, keys, j0, j1;
};
// A CTA's items in turn.  The next one's key count is asked for an item ahead, so that it is not waited for.
struct XItems {
  const XFwdParams& p;
  const XCount by;
  uint32_t i;
  XCount at;
  int keys = 0;
  __device__ __forceinline__ explicit XItems(const XFwdParams& q)
      : p(q), by(x_count(gridDim.x, q.row_tiles, q.splits, q.hv)), i(blockIdx.x),
        at(x_count(blockIdx.x, q.row_tiles, q.splits, q.hv)) {
    if (i < p.items) keys = x_raw_count(p.a, at.d3);
  }
  __device__ __forceinline__ bool next(XItem& t) {
    if (i >= p.items) return false;
    t.tile = at.d0;
    t.split = at.d1;
    t.hv = at.d2;
    t.b = at.d3;
    t.keys = x_key_count(p.a, keys);
    const int n = (t.keys + kXTile - 1) / kXTile;
    t.j0 = min(n, t.split * p.key_chunk);
    t.j1 = min(n, t.j0 + p.key_chunk);
    i += gridDim.x;
    x_advance(at, by, p.row_tiles, p.splits, p.hv);
    if (i < p.items) keys = x_raw_count(p.a, at.d3);
    return true;
  }
};
// 32-key chunks of key tile j that hold keys, and of the 64 keys from u * 64.
__device__ __forceinline__ int x_chunks(int keys, int j) { return (min(kXTile, keys - j * kXTile) + 31) >> 5; }
__device__ __forceinline__ int x_chunks64(int keys, int u) { return (min(64, keys - u * 64) + 31) >> 5; }

// Joins the splits of one warp's rows, in their order: o = sum_s 2^(lse_s - lse) o_s.  For calls of few rows whose splits
// of a (sequence, head group) make up a cluster of one item a CTA: its first CTA joins them when all have met at the
// cluster's barrier, for which no memory is shared with other calls.  Such calls wait for the host, and this saves it a
// launch of x_combine_kernel (one query over 1,024 keys: 11.1 us a call against 13.2).
// r_index: this lane's row; o_at: where its output goes.
template <typename T>
__device__ __forceinline__ void x_join(const XFwdParams& p, bool live, int64_t r_index, int64_t o_at) {
  const int lane = threadIdx.x & 31;
  const int head_dim = p.a.head_dim, rows = __popc(__ballot_sync(~0u, live));  // the first lanes
  // ---- lane = row: the sum of the splits' weights
  constexpr int kAtOnce = 8;
  float m = -INFINITY, total = 0.0f;
  for (int s0 = 0; s0 < p.splits; s0 += kAtOnce) {
    float x[kAtOnce], most = m;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      x[u] = live && s0 + u < p.splits ? __ldcg(p.part_lse + (s0 + u) * p.rows + r_index) : -INFINITY;
      most = fmaxf(most, x[u]);
    }
    const float ref = most == -INFINITY ? 0.0f : most;
    total *= ex2(m - ref);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) total += ex2(x[u] - ref);
    m = most;
  }
  const float ref = m == -INFINITY ? 0.0f : m;
  const float inv = total > 0.0f ? __fdividef(1.0f, total) : (total == total ? 0.0f : total);
  if (p.a.lse != nullptr && live)
    p.a.lse[r_index] = total > 0.0f ? (ref + __log2f(total)) * 0.6931471805599453f : (total == total ? -INFINITY : total);
  // ---- lane = four channels: row after row and split after split, eight loads under way
  const bool mine = lane * 4 < head_dim;
  float acc[4] = {};
  int row = 0, s = 0;  // of the next load, and (to_row, to_s) of the next sum
  int to_row = 0, to_s = 0;
  while (to_row < rows) {
    float4 v[kAtOnce];
    float f[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int64_t at = __shfl_sync(~0u, r_index, row & 31) + s * p.rows;
      f[u] = row < rows ? __ldcg(p.part_lse + at) : -INFINITY;
      v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (mine && row < rows) v[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * head_dim) + lane);
      if (++s == p.splits) {
        s = 0;
        ++row;
      }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (to_row >= rows) break;
      const float w = ex2(f[u] - __shfl_sync(~0u, ref, to_row)) * __shfl_sync(~0u, inv, to_row);
      if (f[u] != -INFINITY) {  // a split without keys wrote no output
        acc[0] = fmaf(w, v[u].x, acc[0]);
        acc[1] = fmaf(w, v[u].y, acc[1]);
        acc[2] = fmaf(w, v[u].z, acc[2]);
        acc[3] = fmaf(w, v[u].w, acc[3]);
      }
      if (++to_s == p.splits) {
        T* const o = static_cast<T*>(p.a.o) + __shfl_sync(~0u, o_at, to_row);
        if (mine)
          *reinterpret_cast<uint2*>(o + lane * 4) =
              make_uint2(XType<T>::pack2(acc[0], acc[1]), XType<T>::pack2(acc[2], acc[3]));
        acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
        to_s = 0;
        ++to_row;
      }
    }
  }
}

template <typename T, int HALVES, bool SPLIT>
__global__ void __launch_bounds__(XFwdLayout<HALVES>::kThreads, kXFwdCtasPerSm)
    x_fwd_kernel(const XFwdParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap o_map) {
  using Ly = XFwdLayout<HALVES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint4* words = reinterpret_cast<uint4*>(smem + Ly::kWords);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + Ly::kBar);
  uint64_t* q_empty = q_full + Ly::kQStages;
  uint64_t* kv_full = q_empty + Ly::kQStages;
  uint64_t* kv_empty = kv_full + Ly::kEntries;
  uint64_t* s_full = kv_empty + Ly::kEntries;  // [2], by score buffer
  uint64_t* p_full = s_full + 2;               // [2]: a warp may be a step ahead of another
  uint64_t* pv_done = p_full + 2;              // [2]: a step's P V product is done
  uint64_t* o_full = pv_done + 2;              // the item's last one is
  uint64_t* o_free = o_full + 1;
  uint64_t* staged = o_free + 1;
  uint64_t* drained = staged + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Ly::kTail);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < Ly::kQStages; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
    }
    for (int i = 0; i < Ly::kEntries; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 2);  // the products' commit, and the issuing thread (keep bits)
      mbar_init(p_full + i, 4);
      mbar_init(pv_done + i, 1);
    }
    mbar_init(o_full, 1);
    mbar_init(o_free, 4);
    mbar_init(staged, 4);
    mbar_init(drained, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == Ly::kWarps) {
    tmem_alloc(tmem_slot, Ly::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  const XAttnParams& a = p.a;
  const bool masked = a.key_mask != nullptr;
  const int ksteps = (a.head_dim + 15) >> 4;  // 16-channel steps of Q K^T, and 16-column steps of P V's width

  if (warp == Ly::kWarps) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      tma_prefetch_desc(&q_map);
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
    }
    const uint32_t q_bytes = static_cast<uint32_t>(a.tile_tokens * a.pack) * 128u * HALVES;
    uint32_t e = 0, loaded = 0, n_item = 0, g = 0;  // `loaded`: entries whose copy was started
    bool ok = true;
    XItems items(p);
    XItem t;
    while (ok && items.next(t)) {
      if (t.j0 >= t.j1) continue;
      const int qs = n_item % Ly::kQStages;
      ok = warp_wait(q_empty + qs, ((n_item / Ly::kQStages) & 1) ^ 1, abort_flag, a.err, kErrXForward + kWaitQFree);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full + qs, q_bytes);
        for (int hf = 0; hf < HALVES; ++hf)
          tma_load_4d(smem + qs * Ly::kTileBytes + hf * 16384, &q_map, q_full + qs, hf * 64, t.hv * a.pack,
                      t.tile * a.tile_tokens, t.b);
      }
      ++n_item;
      const int hk = t.hv * a.pack / a.group;
      for (int j = t.j0; j < t.j1 && ok; ++j, ++g) {
        const bool bits = masked || (j + 1) * kXTile > t.keys;
        if (bits) {
          const uint4 w = x_keep_words(a, t.b, j * kXTile, t.keys, lane);
          if (lane == 0) words[g % kXMaskSlots] = w;
        }
#pragma unroll
        for (int kv = 0; kv < 2 && ok; ++kv, ++e) {
          const int slot = e % Ly::kEntries;
          ok = warp_wait(kv_empty + slot, ((e / Ly::kEntries) & 1) ^ 1, abort_flag, a.err, kErrXForward + kWaitKFree + kv);
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
        mbar_wait(kv_full + k % Ly::kEntries, (k / Ly::kEntries) & 1, &never, a.err, kErrXForward + kWaitDrain);
      for (uint32_t k = n_item > Ly::kQStages ? n_item - Ly::kQStages : 0; k < n_item; ++k)
        mbar_wait(q_full + k % Ly::kQStages, (k / Ly::kQStages) & 1, &never, a.err, kErrXForward + kWaitDrain);
    }
  } else if (warp > Ly::kWarps) {
    // ------------------------------------------------------------ products
    const uint32_t s_base = smem_u32(smem);
    const uint32_t idesc_o = x_idesc<T>(ksteps * 16, 0, 1);
    const uint32_t t_s = tmem, t_o = tmem + 128;
    uint32_t n_item = 0, g = 0, n_s = 0, n_p = 0;  // items, key tiles, scores, weights
    bool ok = true;
    // Entry e (K of key tile e / 2, or its V) has arrived, V with zeros in the rows that are not kept, which their
    // weights of zero would not keep out if they held an infinity.
    // (What K has in those rows only reaches scores that the softmax replaces.)
    const auto entry = [&](uint32_t e, bool bits, int used) {
      const int slot = e % Ly::kEntries;
      if (!warp_wait(kv_full + slot, (e / Ly::kEntries) & 1, abort_flag, a.err, kErrXForward + kWaitK + (e & 1)))
        return false;
      if (bits && (e & 1)) {
        const uint4 w = words[(e >> 1) % kXMaskSlots];
        if ((w.x & w.y & w.z & w.w) != 0xffffffffu)
          x_zero_rows<HALVES>(smem + Ly::kKV + slot * Ly::kTileBytes, w, used, lane);
      }
      return true;
    };
    XItems items(p);
    XItem t;
    while (ok && items.next(t)) {
      if (t.j0 >= t.j1) continue;
      const int qs = n_item % Ly::kQStages;
      ok = warp_wait(q_full + qs, (n_item / Ly::kQStages) & 1, abort_flag, a.err, kErrXForward + kWaitQ);
      const uint64_t sq = k_major_desc(s_base + qs * Ly::kTileBytes);
      const int u_end = min(2 * t.j1, (t.keys + 63) >> 6);  // 64-key steps [2 * j0, u_end)
      const uint32_t g0 = g - t.j0;                         // a key tile's number in the CTA, less its own
      // S of step u over P of step u - 2, whose product was issued before it (products run in their order)
      const auto issue_s = [&](int u) {
        const uint32_t e = 2 * (g0 + (u >> 1));
        const int j = u >> 1;
        if (!(u & 1) && !entry(e, masked || (j + 1) * kXTile > t.keys, x_chunks(t.keys, j) * 32)) return false;
        tc_fence_after();
        if (elect_one()) {
          products_k_major(t_s + (n_s & 1) * 64, sq,
                           k_major_desc(s_base + Ly::kKV + (e % Ly::kEntries) * Ly::kTileBytes + (u & 1) * 8192),
                           x_idesc<T>(x_chunks64(t.keys, u) * 32, 0, 0), ksteps);
          umma_commit(s_full + (n_s & 1));
          mbar_arrive(s_full + (n_s & 1));
          if ((u & 1) || u == u_end - 1) umma_commit(kv_empty + e % Ly::kEntries);
        }
        __syncwarp();
        ++n_s;
        return true;
      };
      ok = ok && issue_s(2 * t.j0) && (2 * t.j0 + 1 >= u_end || issue_s(2 * t.j0 + 1));
      for (int u = 2 * t.j0; u < u_end && ok; ++u) {
        const uint32_t e = 2 * (g0 + (u >> 1)) + 1;
        const int j = u >> 1;
        // O += P V
        if (!(u & 1)) ok = entry(e, masked || (j + 1) * kXTile > t.keys, x_chunks(t.keys, j) * 32);
        ok = ok && warp_wait(p_full + (n_p & 1), (n_p >> 1) & 1, abort_flag, a.err, kErrXForward + kWaitP);
        if (ok && u == 2 * t.j0 && n_item > 0)  // the last item's output has been read
          ok = warp_wait(o_free, (n_item - 1) & 1, abort_flag, a.err, kErrXForward + kWaitAccFree);
        if (!ok) break;
        const uint64_t sv = mn_major_desc(s_base + Ly::kKV + (e % Ly::kEntries) * Ly::kTileBytes + (u & 1) * 8192);
        const uint32_t later = u > 2 * t.j0 ? 1u : 0u, weights = t_s + (n_p & 1) * 64;
        const int steps = 2 * x_chunks64(t.keys, u);
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k)  // a chunk's P lies in the first 16 of its 32 columns, the low part in the others
            if (k < steps) {
              const uint32_t w = weights + (k >> 1) * 32 + (k & 1) * 8;
              umma_f16_ts(t_o, w, sv + k * 128, idesc_o, k > 0 ? 1u : later);
              if (SPLIT) umma_f16_ts(t_o, w + 16, sv + k * 128, idesc_o, 1u);
            }
          umma_commit(pv_done + (n_p & 1));
          if (u == u_end - 1) umma_commit(o_full);
          if ((u & 1) || u == u_end - 1) umma_commit(kv_empty + e % Ly::kEntries);
        }
        __syncwarp();
        ++n_p;
        if (u + 2 < u_end) ok = issue_s(u + 2);
      }
      g += t.j1 - t.j0;
      ++n_item;
    }
    if (!ok && elect_one()) {  // the products in flight end before the tensor memory is freed
      volatile int never = 0;
      umma_commit(drained);
      mbar_wait(drained, 0, &never, a.err, kErrXForward + kWaitDrain);
    }
  } else {
    // ------------------------------------------------------------ softmax: thread = row
    const int quad = warp, row = quad * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t t_s = t_lane, t_o = t_lane + 128;
    const bool flip = a.scale < 0.0f;  // the largest score is the smallest product
    // log2 units; a zero scale keeps a factor that leaves -inf at -inf
    const float c2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-37f);
    const uint64_t c22 = pair2(c2, c2);
    const int rows = a.tile_tokens * a.pack, my_token = row / a.pack, my_head = row % a.pack;
    const bool hands_out = quad == 0 && lane == 0;
    uint32_t n_s = 0, n_item = 0, g = 0;  // 64-key steps, items, key tiles
    int stored = -1;  // Q stage whose output is on its way out
    // The stage is free for a new Q once the output has been read from it; asked for as late as can be.
    const auto release_stored = [&]() {
      if (Ly::kQStages > 1 && stored >= 0 && hands_out) {
        bulk_wait_group_read<0>();
        mbar_arrive(q_empty + stored);
      }
      stored = -1;
    };
    bool ok = true;
    XItems items(p);
    XItem t;
    while (ok && items.next(t)) {
      const int token = t.tile * a.tile_tokens + my_token;
      const bool live = row < rows && token < a.q_len;
      const int head = t.hv * a.pack + my_head;
      const int64_t r_index = (static_cast<int64_t>(t.b) * a.heads + head) * a.q_len + token;
      // rows of this warp that exist: a warp without any keeps only the barriers
      const bool any_row = __any_sync(0xffffffffu, live);
      const int64_t o_at = t.b * a.so.batch + token * a.so.token + head * a.so.head;
      if (t.j0 >= t.j1) {  // no keys
        if (live) {
          if (p.splits > 1) {
            p.part_lse[t.split * p.rows + r_index] = -INFINITY;
          } else {
            T* o = static_cast<T*>(a.o) + o_at;
            for (int c = 0; c < a.head_dim; c += 8) *reinterpret_cast<uint4*>(o + c) = make_uint4(0, 0, 0, 0);
            if (a.lse != nullptr) a.lse[r_index] = -INFINITY;
          }
        }
        continue;
      }
      const int qs = n_item % Ly::kQStages;
      float m = -INFINITY, l = 0.0f;  // reference of the row's exponent, and the sum
      const int u_end = min(2 * t.j1, (t.keys + 63) >> 6);
      for (int u = 2 * t.j0; u < u_end; ++u, ++n_s) {
        const uint32_t scores = t_s + (n_s & 1) * 64;
        ok = warp_wait(s_full + (n_s & 1), (n_s >> 1) & 1, abort_flag, a.err, kErrXForward + kWaitS);
        if (!ok) break;
        tc_fence_after();
        if (any_row) {
          const bool two = x_chunks64(t.keys, u) == 2;
          uint32_t v[2][32];
          tmem_read(scores, v[0]);
          if (two) tmem_read(scores + 32, v[1]);
          if (masked || flip || (u + 1) * 64 > t.keys) {
            uint2 keep = make_uint2(~0u, ~0u);
            if (masked || ((u >> 1) + 1) * kXTile > t.keys)
              keep = reinterpret_cast<const uint2*>(words + (g + (u >> 1) - t.j0) % kXMaskSlots)[u & 1];
            const uint32_t sign = flip ? 0x80000000u : 0u;
#pragma unroll
            for (int k = 0; k < 32; ++k) v[0][k] = (keep.x >> k) & 1u ? v[0][k] ^ sign : 0xff800000u;
            if (two) {
#pragma unroll
              for (int k = 0; k < 32; ++k) v[1][k] = (keep.y >> k) & 1u ? v[1][k] ^ sign : 0xff800000u;
            }
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (c == 0 || two) {
#pragma unroll
              for (int k = 0; k < 32; k += 8)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  mx[i] = max3(mx[i], __uint_as_float(v[c][k + 2 * i]), __uint_as_float(v[c][k + 2 * i + 1]));
            }
          const float mt = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
          // raises the reference where the row's maximum passes it by more than 2^8, with what was summed so far
          if (__any_sync(0xffffffffu, live && ((mt - m) * c2 > 8.0f || m == -INFINITY))) {
            const float mn = fmaxf(m, mt);
            const float f = m == -INFINITY ? 0.0f : ex2((m - mn) * c2);
            l *= f;
            m = mn;
            if (u > 2 * t.j0) {
              // the product of the step before is done (the one before that was when this step's scores came)
              ok = warp_wait(pv_done + ((n_s - 1) & 1), ((n_s - 1) >> 1) & 1, abort_flag, a.err,
                             kErrXForward + kWaitPV);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < 4 * HALVES; ++c) {
                uint32_t o[16];
                tmem_read(t_o + c * 16, o);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                tmem_st_32x32b_x16(t_o + c * 16, o);
              }
            }
          }
          const float mc = m == -INFINITY ? 0.0f : -m * c2;
          const uint64_t mc2 = pair2(mc, mc);
          uint64_t sum[2] = {pair2(0.0f, 0.0f), pair2(0.0f, 0.0f)};
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (c == 0 || two) {
              uint32_t pk[16], lo[16];
#pragma unroll
              for (int k = 0; k < 32; k += 2) {
                float x0, x1;
                unpair2(fma2(pair2(__uint_as_float(v[c][k]), __uint_as_float(v[c][k + 1])), c22, mc2), x0, x1);
                x0 = ex2(x0);
                x1 = ex2(x1);
                sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], pair2(x0, x1));
                if constexpr (SPLIT) split2<T>(x0, x1, pk[k >> 1], lo[k >> 1]);
                else pk[k >> 1] = XType<T>::pack2(x0, x1);
              }
              tmem_st_32x32b_x16(scores + c * 32, pk);  // the weights take the place of their scores
              if constexpr (SPLIT) tmem_st_32x32b_x16(scores + c * 32 + 16, lo);
            }
          float s0, s1;
          unpair2(add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + (n_s & 1));
      }
      if (!ok) break;
      g += t.j1 - t.j0;
      release_stored();
      ok = warp_wait(o_full, n_item & 1, abort_flag, a.err, kErrXForward + kWaitAcc);
      if (!ok) break;
      tc_fence_after();
      const float inv = l > 0.0f ? __fdividef(1.0f, l) : (l == l ? 0.0f : l);
      uint8_t* stage = smem + qs * Ly::kTileBytes;  // Q's tile, read by every product of the item by now
      if (any_row) {
#pragma unroll
        for (int c = 0; c < 2 * HALVES; ++c) {
          const int col = c * 32;
          uint32_t o[32];
          tmem_read(t_o + col, o);
          if (p.splits > 1) {
            if (live) {
              float* dst = p.part_o + (t.split * p.rows + r_index) * a.head_dim + col;
#pragma unroll
              for (int k = 0; k < 32; k += 4)
                if (col + k < a.head_dim)
                  *reinterpret_cast<float4*>(dst + k) =
                      make_float4(__uint_as_float(o[k]) * inv, __uint_as_float(o[k + 1]) * inv,
                                  __uint_as_float(o[k + 2]) * inv, __uint_as_float(o[k + 3]) * inv);
            }
          } else {
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 32; k += 2)
              pk[k >> 1] = XType<T>::pack2(__uint_as_float(o[k]) * inv, __uint_as_float(o[k + 1]) * inv);
#pragma unroll
            for (int u = 0; u < 4; ++u)
              st_shared_v4(stage + (col >> 6) * 16384 + swizzle128_offset(row, ((col & 63) >> 3) + u), pk[4 * u],
                           pk[4 * u + 1], pk[4 * u + 2], pk[4 * u + 3]);
          }
        }
        if (live) {
          // lse in base 2; the natural one is log(2) times it
          const float lse2 = l > 0.0f ? m * c2 + __log2f(l) : (l == l ? -INFINITY : l);
          if (p.splits > 1) p.part_lse[t.split * p.rows + r_index] = lse2;
          else if (a.lse != nullptr) a.lse[r_index] = lse2 * 0.6931471805599453f;
        }
      }
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(staged);
        mbar_arrive(o_free);
      }
      if (hands_out) {
        ok = mbar_wait(staged, n_item & 1, abort_flag, a.err, kErrXForward + kWaitStaged);
        if (ok && p.splits == 1) {
          for (int hf = 0; hf < HALVES; ++hf)
            tma_store_4d(&o_map, stage + hf * 16384, hf * 64, t.hv * a.pack, t.tile * a.tile_tokens, t.b);
          bulk_commit_group();
        }
        if (ok && Ly::kQStages == 1) {
          bulk_wait_group_read<0>();
          mbar_arrive(q_empty + qs);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      stored = qs;
      ++n_item;
    }
    if (hands_out) bulk_wait_group<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == Ly::kWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, Ly::kTmemCols);
  }
  if constexpr (SPLIT) {  // (calls of few rows)
    if (p.join) {
      __syncwarp();
      cluster_sync();
      if (cluster_ctarank() == 0 && warp == 0) {
        const XCount at = x_count(blockIdx.x, p.row_tiles, p.splits, p.hv);
        const int token = lane / a.pack, head = at.d2 * a.pack + lane % a.pack;
        const bool live = lane < a.q_len * a.pack;
        x_join<T>(p, live, (static_cast<int64_t>(at.d3) * a.heads + head) * a.q_len + token,
                  at.d3 * a.so.batch + token * a.so.token + head * a.so.head);
      }
    }
  }
}

// Joins the splits of a row in a launch of its own (see x_join): o = sum_s 2^(lse_s - lse) o_s, in the order of the splits.  One warp per row.
template <typename T>
__global__ void __launch_bounds__(256) x_combine_kernel(const XFwdParams p) {
  pdl_sync();
  const XAttnParams& a = p.a;
  const int lane = threadIdx.x & 31;
  for (int64_t r = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; r < p.rows;
       r += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
    const int token = static_cast<int>(r % a.q_len), head = static_cast<int>(r / a.q_len % a.heads),
              b = static_cast<int>(r / a.q_len / a.heads);
    float w[kXMaxSplits / 32], m = -INFINITY;  // lane = split
#pragma unroll
    for (int k = 0; k < kXMaxSplits / 32; ++k) {
      w[k] = k * 32 + lane < p.splits ? p.part_lse[(k * 32 + lane) * p.rows + r] : -INFINITY;
      m = fmaxf(m, w[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ref = m == -INFINITY ? 0.0f : m;
    float total = 0.0f, o[4] = {};
#pragma unroll
    for (int k = 0; k < kXMaxSplits / 32; ++k) total += w[k] = ex2(w[k] - ref);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    constexpr int kAtOnce = 8;  // loads under way
#pragma unroll
    for (int k = 0; k < kXMaxSplits / 32; ++k)
      for (int s0 = k * 32; s0 < min(p.splits, k * 32 + 32); s0 += kAtOnce) {
        float4 v[kAtOnce];
        float f[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          f[u] = __shfl_sync(0xffffffffu, w[k], (s0 + u) & 31);  // 0 beyond the splits
          v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (f[u] != 0.0f && lane * 4 < a.head_dim)  // a split without keys wrote no output
            v[u] = *reinterpret_cast<const float4*>(p.part_o + ((s0 + u) * p.rows + r) * a.head_dim + lane * 4);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          o[0] = fmaf(f[u], v[u].x, o[0]);
          o[1] = fmaf(f[u], v[u].y, o[1]);
          o[2] = fmaf(f[u], v[u].z, o[2]);
          o[3] = fmaf(f[u], v[u].w, o[3]);
        }
      }
    const float inv = total > 0.0f ? __fdividef(1.0f, total) : (total == total ? 0.0f : total);
    if (lane * 4 < a.head_dim)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + b * a.so.batch + token * a.so.token + head * a.so.head + lane * 4) =
          make_uint2(XType<T>::pack2(o[0] * inv, o[1] * inv), XType<T>::pack2(o[2] * inv, o[3] * inv));
    if (a.lse != nullptr && lane == 0)
      a.lse[r] = total > 0.0f ? (ref + __log2f(total)) * 0.6931471805599453f : (total == total ? -INFINITY : total);
  }
}

}  // namespace fp8b
