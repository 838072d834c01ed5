// host.h — host-side helpers shared by the library's translation units: status and
// error message of the calling thread, per-device state, the tensor-map encoder and
// the kernel launch.  Defined in fp8ops.cu unless they are templates.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

#include "fp8ops.h"

namespace fp8host {

// Records (status, message) for the calling thread and returns the status.
int set_error(int status, const char* fmt, ...);
// Clears the calling thread's status and returns FP8_OK.
int ok();

#define FP8_CUDA_TRY(expr)                                                                       \
  do {                                                                                           \
    cudaError_t e_ = (expr);                                                                     \
    if (e_ != cudaSuccess)                                                                       \
      return set_error(FP8_ERR_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e_),     \
                       __FILE__, __LINE__);                                                      \
  } while (0)

#define FP8_REQUIRE(cond, status, ...)         \
  do {                                         \
    if (!(cond)) return set_error(status, __VA_ARGS__); \
  } while (0)

// Kernels launched through this library since load (graph replays not included).
void count_launches(unsigned n);

struct DeviceState {
  int sm_count = 0;
  int* err_ptr = nullptr;             // device error word
  unsigned int* fold_base = nullptr;  // the device's counters (fold_counter)
  std::atomic<unsigned int> fold_next{0};
  // Set (release) after the fields above are written; a reader that sees it
  // (acquire) sees them too.
  std::atomic<bool> init{false};
};

// The current device's state.
int device_state(DeviceState** out);

// Counters in device memory that a launch's CTAs meet at, zero between launches.
constexpr int kFoldCounters = 8192;
// The counter of the next launch that folds a scale in its last CTA, or holds a grid barrier.
inline unsigned int* fold_counter(DeviceState* st) {
  return st->fold_base + st->fold_next.fetch_add(1, std::memory_order_relaxed) % kFoldCounters;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int get_encode_fn(EncodeTiledFn* out);

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Programmatic dependent launch: 0 = plain stream order (the default), 1 = the
// tensor-core kernels, 2 = every kernel.  Each kernel waits for its predecessor
// (pdl_sync / pdl_wait) before touching global memory, so the attribute only
// lets its CTAs start, and run their prologue, while the previous kernel's CTAs
// drain.  Measured on B200: a conv kernel following another conv kernel gains
// 0.5-1 us, but the quantize -> conv chains of a training step gain nothing
// (their streaming kernels leave no SM free early), so it is off by default.
extern int g_pdl;

enum KernelClass { kStreamingKernel = 0, kTensorKernel = 1 };

// Launch `kern` on `stream`, with programmatic stream serialization when enabled
// for its class, optionally as clusters of `cluster_x` CTAs.
template <typename... KArgs, typename... Args>
cudaError_t launch_kernel(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                          int cluster_x, KernelClass cls, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (g_pdl == 2 || (g_pdl == 1 && cls == kTensorKernel)) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  if (cluster_x > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster_x);
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

}  // namespace fp8host
