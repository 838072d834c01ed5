// conditioning.cu — C ABI of the text-conditioning operators (include/fp8ops.h): the
// token embedding, the counter-based dropout and the attention over an encoder's
// states.  Host code validates, lays out workspaces and launches; it allocates nothing.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "cross_attention.cuh"
#include "cross_attention_bwd.cuh"
#include "dropout.cuh"
#include "embedding.cuh"
#include "fp8ops.h"
#include "host.h"

using namespace fp8b;
using namespace fp8host;

namespace {

cudaStream_t cuda_stream(fp8_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

int dtype_size(int dtype) { return dtype == FP8_DTYPE_FP32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype >= FP8_DTYPE_BF16 && dtype <= FP8_DTYPE_FP16; }

// Calls f with a value of the C++ type of `dtype`.
template <typename F>
int with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case FP8_DTYPE_BF16: return f(__nv_bfloat16{});
    case FP8_DTYPE_FP32: return f(float{});
    default: return f(__half{});
  }
}

unsigned grid_for(int64_t items, int64_t per_block, int sm_count, int blocks_per_sm) {
  const int64_t blocks = (items + per_block - 1) / per_block;
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(blocks, int64_t(sm_count) * blocks_per_sm)));
}

// ------------------------------------------------------------------ cross attention
bool strides_fit(const fp8_head_strides& s, int batch, int tokens, int heads) {
  const auto fits = [](int n, int64_t stride) { return n == 1 || (stride > 0 && stride % 8 == 0); };
  return fits(batch, s.batch) && fits(tokens, s.token) && fits(heads, s.head);
}
XStrides strides_of(const fp8_head_strides& s) { return {s.batch, s.token, s.head}; }

int x_check(const fp8_cross_attention_args* a, bool backward) {
  FP8_REQUIRE(a != nullptr, FP8_ERR_INVALID_ARGUMENT, "cross attention: args is NULL");
  FP8_REQUIRE(a->batch > 0 && a->q_len > 0 && a->k_len > 0 && a->heads > 0 && a->kv_heads > 0,
              FP8_ERR_INVALID_ARGUMENT, "cross attention: sizes must be positive (batch %d, q_len %d, k_len %d, heads %d, "
              "kv_heads %d)", a->batch, a->q_len, a->k_len, a->heads, a->kv_heads);
  // (so that tile and key numbers rounded up stay 32-bit ones)
  FP8_REQUIRE(a->q_len <= INT32_MAX - kXTile && a->k_len <= INT32_MAX - kXTile, FP8_ERR_UNSUPPORTED,
              "cross attention: too long (q_len %d, k_len %d)", a->q_len, a->k_len);
  FP8_REQUIRE(a->heads % a->kv_heads == 0, FP8_ERR_INVALID_ARGUMENT,
              "cross attention: %d heads are not a multiple of %d key heads", a->heads, a->kv_heads);
  FP8_REQUIRE(a->head_dim >= 8 && a->head_dim <= 128 && a->head_dim % 8 == 0, FP8_ERR_UNSUPPORTED,
              "cross attention: head_dim must be a multiple of 8 up to 128, got %d", a->head_dim);
  FP8_REQUIRE(a->dtype == FP8_DTYPE_BF16 || a->dtype == FP8_DTYPE_FP16, FP8_ERR_UNSUPPORTED,
              "cross attention: dtype must be bf16 or fp16, got code %d", a->dtype);
  FP8_REQUIRE(std::isfinite(a->scale), FP8_ERR_INVALID_ARGUMENT, "cross attention: scale is not finite");
  FP8_REQUIRE(a->q && a->k && a->v && a->o && aligned(a->q, 16) && aligned(a->k, 16) && aligned(a->v, 16) &&
                  aligned(a->o, 16) && aligned(a->lse, 4) && aligned(a->key_lengths, 4),
              FP8_ERR_INVALID_ARGUMENT, "cross attention: q, k, v and o must be 16-byte aligned, lse and key_lengths 4-byte");
  FP8_REQUIRE(strides_fit(a->q_stride, a->batch, a->q_len, a->heads) &&
                  strides_fit(a->o_stride, a->batch, a->q_len, a->heads) &&
                  strides_fit(a->k_stride, a->batch, a->k_len, a->kv_heads) &&
                  strides_fit(a->v_stride, a->batch, a->k_len, a->kv_heads),
              FP8_ERR_INVALID_ARGUMENT, "cross attention: strides must be positive multiples of 8 elements");
  if (backward) {
    FP8_REQUIRE(a->lse && a->dout && a->dq && a->dk && a->dv && aligned(a->dout, 16) && aligned(a->dq, 16) &&
                    aligned(a->dk, 16) && aligned(a->dv, 16),
                FP8_ERR_INVALID_ARGUMENT,
                "cross attention backward: needs lse, and dout, dq, dk and dv 16-byte aligned");
    FP8_REQUIRE(strides_fit(a->dout_stride, a->batch, a->q_len, a->heads) &&
                    strides_fit(a->dq_stride, a->batch, a->q_len, a->heads) &&
                    strides_fit(a->dk_stride, a->batch, a->k_len, a->kv_heads) &&
                    strides_fit(a->dv_stride, a->batch, a->k_len, a->kv_heads),
                FP8_ERR_INVALID_ARGUMENT, "cross attention backward: strides must be positive multiples of 8 elements");
  }
  return FP8_OK;
}

XAttnParams x_params(const fp8_cross_attention_args* a, DeviceState* st) {
  XAttnParams p{};
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.o = a->o;
  p.o_in = a->o;
  p.lse = a->lse;
  p.dout = a->dout;
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  p.sq = strides_of(a->q_stride);
  p.sk = strides_of(a->k_stride);
  p.sv = strides_of(a->v_stride);
  p.so = strides_of(a->o_stride);
  p.sdo = strides_of(a->dout_stride);
  p.sdq = strides_of(a->dq_stride);
  p.sdk = strides_of(a->dk_stride);
  p.sdv = strides_of(a->dv_stride);
  p.key_lengths = a->key_lengths;
  p.key_mask = a->key_mask;
  p.mask_stride = a->mask_stride;
  p.batch = a->batch;
  p.q_len = a->q_len;
  p.k_len = a->k_len;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  p.group = a->heads / a->kv_heads;
  p.pack = p.group <= kXTile ? p.group : 1;
  p.tile_tokens = kXTile / p.pack;
  p.scale = a->scale;
  p.err = st->err_ptr;
  return p;
}

// [batch][tokens][heads][channels] of 16-bit values with 64-channel, 128-byte-swizzled
// rows: box {64 channels, box_heads, box_tokens, 1}.  What lies outside reads as zero.
int x_map(CUtensorMap* map, const void* ptr, int dtype, const XStrides& st, int batch, int tokens, int heads,
          int channels, int box_heads, int box_tokens) {
  EncodeTiledFn enc = nullptr;
  if (int s = get_encode_fn(&enc)) return s;
  // the stride of a dimension of one is never used, but has to be a legal one
  const auto bytes = [](int n, int64_t stride) { return static_cast<cuuint64_t>(n == 1 ? 16 : stride * 2); };
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(channels), static_cast<cuuint64_t>(heads),
                        static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(batch)};
  cuuint64_t strides[3] = {bytes(heads, st.head), bytes(tokens, st.token), bytes(batch, st.batch)};
  cuuint32_t box[4] = {64u, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens), 1u};
  cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  const CUresult r = enc(map, dtype == FP8_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  FP8_REQUIRE(r == CUDA_SUCCESS, FP8_ERR_CUDA, "cuTensorMapEncodeTiled(attention [%d][%d][%d][%d]) failed: %d", batch,
              tokens, heads, channels, (int)r);
  return FP8_OK;
}

// Makes the current device's context current to the driver on this thread too (a thread that has made no runtime
// call yet, such as autograd's, has none, and the tensor-map encoder needs one).
int bind_context() {
  int dev = 0;
  FP8_CUDA_TRY(cudaGetDevice(&dev));
  FP8_CUDA_TRY(cudaSetDevice(dev));
  return FP8_OK;
}

// How a forward call divides its work.
struct XPlan {
  int row_tiles, hv, n_tiles, splits, key_chunk;
  int64_t rows, items, slots;
  bool two_values;   // P in two values of the type: x_fwd_kernel's SPLIT
  bool join_inside;  // x_join (with two_values only): the splits are a cluster
};
XPlan x_plan(const fp8_cross_attention_args* a, int sm_count) {
  XPlan w{};
  const int group = a->heads / a->kv_heads, pack = group <= kXTile ? group : 1, tokens = kXTile / pack;
  w.row_tiles = (a->q_len + tokens - 1) / tokens;
  w.hv = a->heads / pack;
  w.n_tiles = (a->k_len + kXTile - 1) / kXTile;
  w.rows = static_cast<int64_t>(a->batch) * a->heads * a->q_len;
  w.slots = static_cast<int64_t>(sm_count) * kXFwdCtasPerSm;
  const int64_t base = static_cast<int64_t>(a->batch) * w.hv * w.row_tiles;
  w.splits = 1;
  w.key_chunk = w.n_tiles;
  // A split writes its rows' partial outputs in fp32.  With a few rows a tile that is nothing, and pieces that are a
  // quarter of an even share even out sequences of different lengths (finer ones only make the join longer: 32 queries
  // over 8192 keys, with their weights rounded once 88 us and the join at four pieces a CTA, the same at eight and
  // twelve, 92 at sixteen).  With whole
  // tiles of rows the keys are split only to reach SMs that would have no work at all (5 x 333 queries of 8 heads over
  // 1021 keys, 110 row tiles: 28 us unsplit, 36 split for two CTAs an SM).
  const bool few_rows = w.row_tiles == 1 && a->q_len * pack <= 16;
  const int64_t pieces = few_rows ? 4 * w.slots : sm_count;
  if (w.n_tiles > 1 && 2 * base <= pieces) {
    w.key_chunk = static_cast<int>(std::max<int64_t>((w.n_tiles * base + pieces - 1) / pieces,
                                                     (w.n_tiles + kXMaxSplits - 1) / kXMaxSplits));
    w.splits = (w.n_tiles + w.key_chunk - 1) / w.key_chunk;
  }
  w.two_values = w.n_tiles == 1 || few_rows;
  // Joined by the launch itself where the splits fit a cluster of the portable sizes 2, 4 and 8 (the last ones may have no
  // keys) and every CTA has one item: a CTA that goes on with other items would be held up.  (Joined at counters in
  // memory, zeroed before the launch: 12.3 us for one query of 4 heads of 64 over 1,024 keys, 30.8 over 8,192, whose 64
  // splits take 22.5 with a second launch; in a cluster 11.1.)
  int cluster = 2;
  while (cluster < w.splits) cluster *= 2;
  w.join_inside = few_rows && w.splits > 1 && cluster <= 8 && base * cluster <= w.slots;
  if (w.join_inside) w.splits = cluster;
  w.items = base * w.splits;
  return w;
}
// The workspace: the splits' outputs and their log-sum-exps.
size_t x_fwd_workspace(const fp8_cross_attention_args* a, const XPlan& w) {
  return w.splits == 1 ? 0 : sizeof(float) * static_cast<size_t>(w.splits) * w.rows * (a->head_dim + 1);
}

template <typename T, int HALVES>
int x_fwd_launch(const XFwdParams& f, const CUtensorMap (&maps)[4], bool two_values, int64_t slots, cudaStream_t stream) {
  using Ly = XFwdLayout<HALVES>;
  const auto kernel = two_values ? x_fwd_kernel<T, HALVES, true> : x_fwd_kernel<T, HALVES, false>;
  FP8_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Ly::kSmemBytes));
  FP8_CUDA_TRY(launch_kernel(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(f.items, slots))), dim3(Ly::kThreads),
                             Ly::kSmemBytes, stream, f.join ? f.splits : 1, kTensorKernel, f, maps[0], maps[1], maps[2],
                             maps[3]));
  count_launches(1);
  return FP8_OK;
}

template <typename T>
int x_fwd(const fp8_cross_attention_args* args, const XAttnParams& a, const XPlan& w, void* workspace, DeviceState* st,
          cudaStream_t stream) {
  XFwdParams f{};
  f.a = a;
  f.row_tiles = w.row_tiles;
  f.hv = w.hv;
  f.key_chunk = w.key_chunk;
  f.splits = w.splits;
  f.part_o = static_cast<float*>(workspace);
  f.part_lse = f.part_o == nullptr ? nullptr : f.part_o + static_cast<int64_t>(w.splits) * w.rows * a.head_dim;
  f.rows = w.rows;
  f.items = static_cast<uint32_t>(w.items);
  if (int s = bind_context()) return s;
  f.join = w.join_inside;
  CUtensorMap maps[4];
  const int dt = args->dtype;
  if (int s = x_map(&maps[0], a.q, dt, a.sq, a.batch, a.q_len, a.heads, a.head_dim, a.pack, a.tile_tokens)) return s;
  if (int s = x_map(&maps[1], a.k, dt, a.sk, a.batch, a.k_len, a.kv_heads, a.head_dim, 1, kXTile)) return s;
  if (int s = x_map(&maps[2], a.v, dt, a.sv, a.batch, a.k_len, a.kv_heads, a.head_dim, 1, kXTile)) return s;
  if (int s = x_map(&maps[3], a.o, dt, a.so, a.batch, a.q_len, a.heads, a.head_dim, a.pack, a.tile_tokens)) return s;
  const int status = a.head_dim <= 64 ? x_fwd_launch<T, 1>(f, maps, w.two_values, w.slots, stream)
                                      : x_fwd_launch<T, 2>(f, maps, w.two_values, w.slots, stream);
  if (status) return status;
  if (w.splits > 1 && !w.join_inside) {
    FP8_CUDA_TRY(launch_kernel(x_combine_kernel<T>, dim3(grid_for(w.rows, 8, st->sm_count, 8)), dim3(256), 0, stream, 1,
                               kStreamingKernel, f));
    count_launches(1);
  }
  return ok();
}

// How a backward call divides the dK / dV work, and what it keeps in the workspace.
struct XBwdPlan {
  int row_tiles, q_tiles, q_chunk, splits;
  int64_t dq_items, dkv_items;
  size_t stats_bytes, part_bytes, row_norm_bytes, max_norm_bytes;  // the workspace, in this order; the norms for fp16
  size_t bytes() const { return stats_bytes + part_bytes + row_norm_bytes + max_norm_bytes; }
};
XBwdPlan x_bwd_plan(const fp8_cross_attention_args* a, int sm_count) {
  const XPlan f = x_plan(a, sm_count);
  XBwdPlan w{};
  const int group = a->heads / a->kv_heads, pack = a->heads / f.hv;
  w.row_tiles = f.row_tiles;
  w.q_tiles = group / pack * f.row_tiles;
  w.dq_items = static_cast<int64_t>(a->batch) * f.hv * f.row_tiles;
  const int64_t base = static_cast<int64_t>(a->batch) * a->kv_heads * f.n_tiles;
  // queries are split (and the partial sums joined) only where key tiles alone leave half the SMs without work
  w.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(w.q_tiles, sm_count / base)));
  w.q_chunk = (w.q_tiles + w.splits - 1) / w.splits;
  w.splits = (w.q_tiles + w.q_chunk - 1) / w.q_chunk;
  w.dkv_items = base * w.splits;
  w.stats_bytes = static_cast<size_t>(w.dq_items) * 2 * kXTile * sizeof(float);
  w.part_bytes = w.splits == 1 ? 0 : sizeof(float) * 2 * w.splits * a->batch * a->k_len * static_cast<size_t>(a->kv_heads) * a->head_dim;
  const bool norms = a->dtype == FP8_DTYPE_FP16;
  w.row_norm_bytes = norms ? sizeof(float) * f.rows : 0;
  w.max_norm_bytes = norms ? sizeof(unsigned int) * 2 * a->batch * a->kv_heads : 0;
  return w;
}

template <typename T, int HALVES, bool SPLIT>
int x_bwd_launch(const XBwdParams& dq, const XBwdParams& dkv, const CUtensorMap (&m)[7], DeviceState* st,
                 cudaStream_t stream) {
  FP8_CUDA_TRY(cudaFuncSetAttribute(x_dq_kernel<T, HALVES, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    XDqLayout<HALVES, SPLIT>::kSmemBytes));
  FP8_CUDA_TRY(cudaFuncSetAttribute(x_dkv_kernel<T, HALVES, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    XDkvLayout<HALVES>::kSmemBytes));
  const auto grid = [&](int64_t items) { return dim3(static_cast<unsigned>(std::min<int64_t>(items, st->sm_count))); };
  FP8_CUDA_TRY(launch_kernel(x_dq_kernel<T, HALVES, SPLIT>, grid(dq.items), dim3(kXBwdThreads),
                             XDqLayout<HALVES, SPLIT>::kSmemBytes, stream, 1, kTensorKernel, dq, m[0], m[1], m[2], m[3], m[4]));
  FP8_CUDA_TRY(launch_kernel(x_dkv_kernel<T, HALVES, SPLIT>, grid(dkv.items), dim3(kXBwdThreads),
                             XDkvLayout<HALVES>::kSmemBytes, stream, 1, kTensorKernel, dkv, m[0], m[1], m[2], m[3], m[5],
                             m[6]));
  count_launches(2);
  return FP8_OK;
}

template <typename T>
int x_bwd(const fp8_cross_attention_args* args, const XAttnParams& a, const XBwdPlan& w, void* workspace,
          DeviceState* st, cudaStream_t stream) {
  XBwdParams p{};
  p.a = a;
  p.row_tiles = w.row_tiles;
  p.hv = a.heads / a.pack;
  p.stats = static_cast<float*>(workspace);
  p.items = static_cast<uint32_t>(w.dq_items);
  p.row_norm2 = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.stats_bytes + w.part_bytes);
  p.max_norm2 = reinterpret_cast<unsigned int*>(reinterpret_cast<char*>(p.row_norm2) + w.row_norm_bytes);
  XBwdParams kv = p;
  kv.items = static_cast<uint32_t>(w.dkv_items);
  kv.q_tiles = w.q_tiles;
  kv.q_chunk = w.q_chunk;
  kv.splits = w.splits;
  kv.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.stats_bytes);
  if (int s = bind_context()) return s;
  CUtensorMap m[7];
  const int dt = args->dtype;
  const auto q_side = [&](CUtensorMap* map, const void* ptr, const XStrides& s) {
    return x_map(map, ptr, dt, s, a.batch, a.q_len, a.heads, a.head_dim, a.pack, a.tile_tokens);
  };
  const auto k_side = [&](CUtensorMap* map, const void* ptr, const XStrides& s) {
    return x_map(map, ptr, dt, s, a.batch, a.k_len, a.kv_heads, a.head_dim, 1, kXTile);
  };
  if (int s = q_side(&m[0], a.q, a.sq)) return s;
  if (int s = k_side(&m[1], a.k, a.sk)) return s;
  if (int s = k_side(&m[2], a.v, a.sv)) return s;
  if (int s = q_side(&m[3], a.dout, a.sdo)) return s;
  if (int s = q_side(&m[4], a.dq, a.sdq)) return s;
  if (int s = k_side(&m[5], a.dk, a.sdk)) return s;
  if (int s = k_side(&m[6], a.dv, a.sdv)) return s;
  if constexpr (kXScaled<T>) {
    FP8_CUDA_TRY(cudaMemsetAsync(p.max_norm2, 0, w.max_norm_bytes, stream));
    const int64_t chunks = (static_cast<int64_t>(a.q_len) * a.group + a.k_len + kXNormRows - 1) / kXNormRows * a.batch * a.kv_heads;
    FP8_CUDA_TRY(launch_kernel(x_norms_kernel<T>, dim3(grid_for(chunks, 1, st->sm_count, 8)), dim3(256), 0, stream, 1,
                               kStreamingKernel, p));
    count_launches(1);
  }
  const bool one = a.k_len <= kXTile;  // the states are one key tile
  const int status = a.head_dim <= 64 ? (one ? x_bwd_launch<T, 1, true>(p, kv, m, st, stream)
                                             : x_bwd_launch<T, 1, false>(p, kv, m, st, stream))
                                      : (one ? x_bwd_launch<T, 2, true>(p, kv, m, st, stream)
                                             : x_bwd_launch<T, 2, false>(p, kv, m, st, stream));
  if (status) return status;
  if (w.splits > 1) {
    const int64_t quads = 2ll * a.batch * a.k_len * a.kv_heads * (a.head_dim / 4);
    FP8_CUDA_TRY(launch_kernel(x_dkv_join_kernel<T>, dim3(grid_for(quads, 256, st->sm_count, 8)), dim3(256), 0, stream, 1,
                               kStreamingKernel, kv));
    count_launches(1);
  }
  return ok();
}

}  // namespace

extern "C" {

size_t fp8_cross_attention_workspace_bytes(const fp8_cross_attention_args* a, int backward) {
  DeviceState* st = nullptr;
  if (a == nullptr || a->batch <= 0 || a->q_len <= 0 || a->k_len <= 0 || a->heads <= 0 || a->kv_heads <= 0 ||
      a->heads % a->kv_heads != 0)
    return 0;
  if (device_state(&st)) return 0;
  if (backward) {
    const XBwdPlan w = x_bwd_plan(a, st->sm_count);
    return w.bytes();
  }
  return x_fwd_workspace(a, x_plan(a, st->sm_count));
}

int fp8_cross_attention_fwd(const fp8_cross_attention_args* a, void* workspace, size_t workspace_bytes,
                            fp8_stream_t stream) {
  if (int s = x_check(a, false)) return s;
  DeviceState* st = nullptr;
  if (int s = device_state(&st)) return s;
  const XPlan w = x_plan(a, st->sm_count);
  FP8_REQUIRE(w.items < (1ll << 31), FP8_ERR_UNSUPPORTED, "cross attention: too many row tiles (%lld)", (long long)w.items);
  const size_t need = x_fwd_workspace(a, w);
  FP8_REQUIRE(need == 0 || (workspace != nullptr && aligned(workspace, 16) && workspace_bytes >= need),
              FP8_ERR_WORKSPACE, "cross attention: workspace too small or not 16-byte aligned (%zu bytes, needs %zu)",
              workspace_bytes, need);
  const XAttnParams p = x_params(a, st);
  return a->dtype == FP8_DTYPE_BF16 ? x_fwd<__nv_bfloat16>(a, p, w, workspace, st, cuda_stream(stream))
                                    : x_fwd<__half>(a, p, w, workspace, st, cuda_stream(stream));
}

int fp8_cross_attention_bwd(const fp8_cross_attention_args* a, void* workspace, size_t workspace_bytes,
                            fp8_stream_t stream) {
  if (int s = x_check(a, true)) return s;
  DeviceState* st = nullptr;
  if (int s = device_state(&st)) return s;
  const XBwdPlan w = x_bwd_plan(a, st->sm_count);
  FP8_REQUIRE(w.dq_items < (1ll << 31) && w.dkv_items < (1ll << 31), FP8_ERR_UNSUPPORTED,
              "cross attention backward: too many tiles (%lld, %lld)", (long long)w.dq_items, (long long)w.dkv_items);
  const size_t need = w.bytes();
  FP8_REQUIRE(workspace != nullptr && aligned(workspace, 16) && workspace_bytes >= need, FP8_ERR_WORKSPACE,
              "cross attention backward: workspace too small or not 16-byte aligned (%zu bytes, needs %zu)",
              workspace_bytes, need);
  const XAttnParams p = x_params(a, st);
  return a->dtype == FP8_DTYPE_BF16 ? x_bwd<__nv_bfloat16>(a, p, w, workspace, st, cuda_stream(stream))
                                    : x_bwd<__half>(a, p, w, workspace, st, cuda_stream(stream));
}

// ------------------------------------------------------------------ token embedding
namespace {

// How an embedding gradient is sorted and summed, and where its workspace lies.  By sizes alone: the order of
// the sums, and so the result, does not depend on the device.
struct EmbedPlan {
  int passes, bits, ctas, per_cta;
  int chunk, slices;
  int64_t chunks;
  size_t key[2], pos[2], counts, live, arrive, present, head, tail, bytes;
};
EmbedPlan embed_plan(int64_t tokens, int64_t vocab, int width) {
  EmbedPlan w{};
  int need = 1;  // keys are 0 .. vocab
  while ((int64_t(1) << need) <= vocab) ++need;
  w.passes = (need + kSortMaxBits - 1) / kSortMaxBits;
  w.bits = (need + w.passes - 1) / w.passes;
  // One CTA, without barriers between CTAs, up to 2048 tokens; then 1024 a CTA, one step of each of its warps, while
  // there are CTAs: a step of 32 tokens takes its warp about 100 instructions, and 32 warps share an SM's issue.
  w.ctas = tokens <= 2048 ? 1 : static_cast<int>(std::min<int64_t>(kSortMaxCtas, (tokens + kSortThreads - 1) / kSortThreads));
  w.per_cta = static_cast<int>((tokens + w.ctas * int64_t(kSortThreads) - 1) / (w.ctas * int64_t(kSortThreads))) * kSortThreads;
  w.slices = (width + kSumSlice - 1) / kSumSlice;
  // about 2048 chunks of a slice, of 16 tokens at least: enough warps, and few partial sums of a frequent row
  w.chunk = static_cast<int>(std::max<int64_t>(16, (tokens + 2047) / 2048));
  w.chunks = (tokens + w.chunk - 1) / w.chunk;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 15) & ~size_t(15);
    return here;
  };
  for (int i = 0; i < 2; ++i) {
    w.key[i] = take(sizeof(uint32_t) * static_cast<size_t>(tokens));
    w.pos[i] = take(sizeof(uint32_t) * static_cast<size_t>(tokens));
  }
  w.counts = take(sizeof(uint32_t) * static_cast<size_t>(w.ctas) << w.bits);
  // zeroed before the sort: the number of live keys, and the counter where its CTAs meet.  (The call's own: neither
  // another call nor a replay of a captured one can meet there, and a launch that gave up leaves nothing behind.)
  w.live = take(sizeof(uint32_t));
  w.arrive = take(sizeof(uint32_t));
  w.present = take(sizeof(uint32_t) * static_cast<size_t>(vocab / 32 + 1));
  w.head = take(sizeof(float) * static_cast<size_t>(w.chunks) * width);
  w.tail = take(sizeof(float) * static_cast<size_t>(w.chunks) * width);
  w.bytes = at;
  return w;
}

// The sort's waits: fp8_selftest_sort_timeout.
std::atomic<uint64_t> g_sort_limit_ns{FP8_WAIT_TIMEOUT_NS};
std::atomic<unsigned int> g_sort_missing{0};

// embed_few_kernel takes the gradient: see kFewTokens (and its grid stays small).
bool embed_few(int64_t tokens, int width) {
  return tokens <= kFewTokens && tokens * ((width + kSumSlice - 1) / kSumSlice) <= 1 << 16;
}

}  // namespace

static int embed_check(const void* ids, int ids64, int64_t tokens, int64_t vocab, int width, int weight_dtype,
                       int out_dtype) {
  FP8_REQUIRE(tokens >= 0 && vocab > 0 && width > 0, FP8_ERR_INVALID_ARGUMENT,
              "embedding: bad sizes (tokens %lld, vocab %lld, width %d)", (long long)tokens, (long long)vocab, width);
  FP8_REQUIRE(width <= INT32_MAX - 1024, FP8_ERR_UNSUPPORTED, "embedding: rows too wide (%d)", width);  // (as above)
  FP8_REQUIRE(known_dtype(weight_dtype) && known_dtype(out_dtype), FP8_ERR_UNSUPPORTED,
              "embedding: unknown dtype code %d / %d", weight_dtype, out_dtype);
  FP8_REQUIRE(tokens == 0 || (ids != nullptr && aligned(ids, ids64 ? 8 : 4)), FP8_ERR_INVALID_ARGUMENT,
              "embedding: ids is NULL or misaligned");
  return FP8_OK;
}

int fp8_embedding_fwd(const void* ids, int ids64, int64_t tokens, const void* weight, int weight_dtype, int64_t vocab,
                      int width, int64_t weight_stride, float scale, void* out, int out_dtype, fp8_stream_t stream) {
  if (int s = embed_check(ids, ids64, tokens, vocab, width, weight_dtype, out_dtype)) return s;
  if (tokens == 0) return ok();
  FP8_REQUIRE(weight && out && aligned(weight, dtype_size(weight_dtype)) && aligned(out, dtype_size(out_dtype)),
              FP8_ERR_INVALID_ARGUMENT, "embedding: weight or out is NULL or misaligned");
  DeviceState* st = nullptr;
  if (int s = device_state(&st)) return s;
  EmbedParams p{};
  p.ids = ids;
  p.ids64 = ids64;
  p.weight = weight;
  p.weight_stride = weight_stride;
  p.out = out;
  p.tokens = tokens;
  p.vocab = vocab;
  p.width = width;
  p.scale = scale;
  p.err = st->err_ptr;
  const bool vec = width % 8 == 0 && weight_stride % 8 == 0 && aligned(weight, 16) && aligned(out, 16);
  const int status = with_dtype(weight_dtype, [&](auto w) {
    return with_dtype(out_dtype, [&](auto o) {
      using TW = decltype(w);
      using TO = decltype(o);
      FP8_CUDA_TRY(launch_kernel(vec ? embed_fwd_kernel<TW, TO, true> : embed_fwd_kernel<TW, TO, false>,
                                 dim3(grid_for(tokens, 8, st->sm_count, 8)), dim3(256), 0, cuda_stream(stream), 1,
                                 kStreamingKernel, p));
      return FP8_OK;
    });
  });
  if (status) return status;
  count_launches(1);
  return ok();
}

size_t fp8_embedding_bwd_workspace_bytes(int64_t tokens, int64_t vocab, int width) {
  if (tokens < 0 || vocab <= 0 || width <= 0) return 0;
  return embed_few(tokens, width) ? 0 : embed_plan(tokens, vocab, width).bytes;
}

int fp8_embedding_bwd(const void* ids, int ids64, int64_t tokens, const void* dout, int out_dtype, void* dweight,
                      int weight_dtype, int64_t vocab, int width, float scale, int64_t padding_idx, void* workspace,
                      size_t workspace_bytes, fp8_stream_t stream) {
  if (int s = embed_check(ids, ids64, tokens, vocab, width, weight_dtype, out_dtype)) return s;
  FP8_REQUIRE((tokens == 0 || dout) && dweight && aligned(dweight, dtype_size(weight_dtype)) &&
                  aligned(dout, dtype_size(out_dtype)),
              FP8_ERR_INVALID_ARGUMENT, "embedding backward: dout or dweight is NULL or misaligned");
  FP8_REQUIRE(tokens < (1ll << 31) - (1 << 20) && vocab < (1ll << 31) - 1, FP8_ERR_UNSUPPORTED,
              "embedding backward: too many tokens (%lld) or rows (%lld)", (long long)tokens, (long long)vocab);
  DeviceState* st = nullptr;
  if (int s = device_state(&st)) return s;
  const bool vec = width % 8 == 0 && aligned(dout, 16) && aligned(dweight, 16);
  if (embed_few(tokens, width)) {
    EmbedFewParams f{};
    f.ids = ids;
    f.ids64 = ids64;
    f.tokens = static_cast<int>(tokens);
    f.dout = dout;
    f.dweight = dweight;
    f.vocab = vocab;
    f.padding_idx = padding_idx;
    f.slices = (width + kSumSlice - 1) / kSumSlice;
    f.width = width;
    f.zero_ctas = static_cast<int>(grid_for(vocab, kFewRows, st->sm_count, 8));
    f.scale = scale;
    const int status = with_dtype(weight_dtype, [&](auto wt) {
      return with_dtype(out_dtype, [&](auto o) {
        using TW = decltype(wt);
        using TO = decltype(o);
        FP8_CUDA_TRY(launch_kernel(vec ? embed_few_kernel<TW, TO, true> : embed_few_kernel<TW, TO, false>,
                                   dim3(static_cast<unsigned>(f.zero_ctas + f.tokens * f.slices)), dim3(kFewThreads), 0,
                                   cuda_stream(stream), 1, kStreamingKernel, f));
        return FP8_OK;
      });
    });
    if (status) return status;
    count_launches(1);
    return ok();
  }
  const EmbedPlan w = embed_plan(tokens, vocab, width);
  FP8_REQUIRE(workspace != nullptr && aligned(workspace, 16) && workspace_bytes >= w.bytes, FP8_ERR_WORKSPACE,
              "embedding backward: workspace too small or not 16-byte aligned (%zu bytes, needs %zu)", workspace_bytes,
              w.bytes);
  char* const ws = static_cast<char*>(workspace);
  EmbedSortParams so{};
  so.ids = ids;
  so.ids64 = ids64;
  so.vocab = vocab;
  so.padding_idx = padding_idx;
  so.tokens = static_cast<int>(tokens);
  so.passes = w.passes;
  so.bits = w.bits;
  so.per_cta = w.per_cta;
  so.per_warp = w.per_cta / kSortWarps;
  for (int i = 0; i < 2; ++i) {
    so.key[i] = reinterpret_cast<uint32_t*>(ws + w.key[i]);
    so.pos[i] = reinterpret_cast<uint32_t*>(ws + w.pos[i]);
  }
  so.counts = reinterpret_cast<uint32_t*>(ws + w.counts);
  so.live = reinterpret_cast<uint32_t*>(ws + w.live);
  so.present = reinterpret_cast<uint32_t*>(ws + w.present);
  so.arrive = reinterpret_cast<unsigned int*>(ws + w.arrive);
  so.meet = static_cast<unsigned int>(w.ctas) + g_sort_missing.load(std::memory_order_relaxed);
  so.limit_ns = g_sort_limit_ns.load(std::memory_order_relaxed);
  if (so.meet > 1)  // (one CTA waits for none, and always says how many keys are live)
    FP8_CUDA_TRY(cudaMemsetAsync(so.live, 0, w.arrive + sizeof(uint32_t) - w.live, cuda_stream(stream)));
  so.err = st->err_ptr;
  const size_t smem = sizeof(uint32_t) * ((kSortWarps + 1) * (size_t(1) << w.bits) + kSortWarps);
  FP8_CUDA_TRY(cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(w.ctas));
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = cuda_stream(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;  // the CTAs meet between the passes: all resident
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = w.ctas > 1 ? 1u : 0u;
  FP8_CUDA_TRY(cudaLaunchKernelEx(&cfg, embed_sort_kernel, so));

  EmbedSumParams su{};
  su.key = so.key[(w.passes + 1) & 1];
  su.pos = so.pos[(w.passes + 1) & 1];
  su.live = so.live;
  su.present = so.present;
  su.dout = dout;
  su.dweight = dweight;
  su.head = reinterpret_cast<float*>(ws + w.head);
  su.tail = reinterpret_cast<float*>(ws + w.tail);
  su.vocab = vocab;
  su.chunk = w.chunk;
  su.slices = w.slices;
  su.width = width;
  su.scale = scale;
  const int64_t joins = w.chunks * w.slices;
  const int status = with_dtype(weight_dtype, [&](auto wt) {
    using TW = decltype(wt);
    const int s = with_dtype(out_dtype, [&](auto o) {
      using TO = decltype(o);
      FP8_CUDA_TRY(launch_kernel(vec ? embed_sum_kernel<TW, TO, true> : embed_sum_kernel<TW, TO, false>,
                                 dim3(grid_for(std::max(joins, vocab / 8 + 1), 8, st->sm_count, 8)), dim3(256), 0,
                                 cuda_stream(stream), 1, kStreamingKernel, su));
      return FP8_OK;
    });
    if (s || joins == 0) return s;
    FP8_CUDA_TRY(launch_kernel(embed_join_kernel<TW>, dim3(grid_for(2 * joins, 8, st->sm_count, 8)), dim3(256), 0,
                               cuda_stream(stream), 1, kStreamingKernel, su));
    return FP8_OK;
  });
  if (status) return status;
  count_launches(joins > 0 ? 3 : 2);
  return ok();
}

int fp8_selftest_sort_timeout(uint64_t limit_ns) {
  FP8_REQUIRE(limit_ns <= 1000000000ull, FP8_ERR_INVALID_ARGUMENT, "limit_ns must be at most 1e9");
  g_sort_missing.store(limit_ns == 0 ? 0u : 1u, std::memory_order_relaxed);
  g_sort_limit_ns.store(limit_ns == 0 ? FP8_WAIT_TIMEOUT_NS : limit_ns, std::memory_order_relaxed);
  return ok();
}

// ------------------------------------------------------------------ dropout
int fp8_dropout(const void* x, const void* residual, void* y, int dtype, int64_t n, double p, const int64_t* seed,
                fp8_stream_t stream) {
  FP8_REQUIRE(n >= 0, FP8_ERR_INVALID_ARGUMENT, "dropout: negative size");
  FP8_REQUIRE(known_dtype(dtype), FP8_ERR_UNSUPPORTED, "dropout: unknown dtype code %d", dtype);
  FP8_REQUIRE(p >= 0.0 && p <= 1.0, FP8_ERR_INVALID_ARGUMENT, "dropout: p must be in [0, 1], got %g", p);
  if (n == 0) return ok();
  const size_t size = dtype_size(dtype);
  FP8_REQUIRE(x && y && seed && aligned(x, size) && aligned(y, size) && aligned(residual, size) && aligned(seed, 8),
              FP8_ERR_INVALID_ARGUMENT, "dropout: x, y or seed is NULL, or a pointer is misaligned");
  DeviceState* st = nullptr;
  if (int s = device_state(&st)) return s;
  DropoutParams d{};
  d.x = x;
  d.residual = residual;
  d.y = y;
  d.seed = seed;
  d.n = n;
  d.thresh = static_cast<uint32_t>(std::lrint(p * 65536.0));
  d.scale = p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.0f;
  const int status = with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const bool vec = aligned(x, 16) && aligned(y, 16) && aligned(residual, 16);
    const auto kernel = residual ? (vec ? dropout_kernel<T, true, true> : dropout_kernel<T, false, true>)
                                 : (vec ? dropout_kernel<T, true, false> : dropout_kernel<T, false, false>);
    FP8_CUDA_TRY(launch_kernel(kernel, dim3(grid_for(n, 8 * kDropoutThreads, st->sm_count, 8)), dim3(kDropoutThreads), 0,
                               cuda_stream(stream), 1, kStreamingKernel, d));
    return FP8_OK;
  });
  if (status) return status;
  count_launches(1);
  return ok();
}

}  // extern "C"
