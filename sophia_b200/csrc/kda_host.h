// Host-side helpers shared by the translation units of the library: the
// calling thread's last error, buffer carving, per-launch timing.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <mutex>
#include <string>
#include <vector>

#include "../../include/kda_b200.h"

namespace kda {

inline thread_local std::string g_last_error;

inline int fail(int code, const std::string& msg) {
  g_last_error = msg;
  return code;
}

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Sub-buffer carving of a caller buffer.
struct Carver {
  char* base;
  size_t off = 0;
  explicit Carver(void* p) : base(static_cast<char*>(p)) {}
  template <typename T>
  T* take(size_t bytes) {
    T* p = base ? reinterpret_cast<T*>(base + off) : nullptr;
    off += align256(bytes);
    return p;
  }
};

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// ---- optional per-launch device timing (CUDA events on the launch stream)
enum KernelId {
  K_TABLE = 0, K_FWD_INTRA, K_FWD_STATE, K_BWD_STATE, K_BWD_INTRA, K_BWD_POST, K_REDUCE, K_RECURRENT,
  K_GNORM_FWD, K_GNORM_BWD, K_F32_PREP, K_F32_FWD, K_F32_BWD, K_F32_DC, K_F32_CONV, K_DOC_BOUNDS,
  K_CONV_FWD, K_CONV_BWD, K_CONV_STEP, K_SCAN_FWD, K_SCAN_BWD, K_SCAN_STEP, K_GRAD_NORM, K_GRAD_SCALE,
  K_REC_FWD, K_REC_BWD, K_REC_STEP, K_NORM_FWD, K_NORM_BWD, K_COUNT
};
inline const char* const kKernelNames[K_COUNT] = {"chunk_table", "fwd_intra", "fwd_state",       "bwd_state",
                                           "bwd_intra",   "bwd_post",  "reduce",          "recurrent",
                                           "gated_norm_fwd", "gated_norm_bwd", "f32_prep", "f32_fwd",
                                           "f32_bwd",     "f32_dc",    "f32_conv_bwd",    "doc_bounds",
                                           "conv_fwd",    "conv_bwd",  "conv_step",       "scan_fwd",
                                           "scan_bwd",    "scan_step", "grad_norm",       "grad_scale",
                                           "rec_fwd",     "rec_bwd",   "rec_step",        "norm_fwd",
                                           "norm_bwd"};

struct Timing {
  std::mutex mu;
  bool on = false;
  std::vector<cudaEvent_t> pool;  // pairs (start, stop)
  std::vector<int> ids;           // kernel id of each recorded pair
  size_t used = 0;
};
inline Timing g_timing;

struct TimedLaunch {
  cudaEvent_t stop = nullptr;
  cudaStream_t st;
  TimedLaunch(int id, cudaStream_t s) : st(s) {
    if (!g_timing.on) return;
    std::lock_guard<std::mutex> lk(g_timing.mu);
    if (g_timing.used + 2 > g_timing.pool.size()) {
      for (int i = 0; i < 64; ++i) {
        cudaEvent_t e;
        if (cudaEventCreate(&e) != cudaSuccess) return;
        g_timing.pool.push_back(e);
      }
    }
    cudaEvent_t start = g_timing.pool[g_timing.used];
    stop = g_timing.pool[g_timing.used + 1];
    g_timing.used += 2;
    g_timing.ids.push_back(id);
    cudaEventRecord(start, st);
  }
  ~TimedLaunch() {
    if (stop) cudaEventRecord(stop, st);
  }
};

inline int launch_check(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(KDA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return KDA_OK;
}

// SMs of the current device (queried once per device).
inline int sm_count() {
  static std::atomic<int> counts[64];  // zero-initialised (static storage); concurrent first calls store the same value
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = counts[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
  counts[dev].store(n, std::memory_order_relaxed);
  return n;
}

// Address of the device-side failure flag (kda_b200_device_error) on the
// current device, for the translation units that do not define it; null on
// failure.  Defined in kda_api.cu.
int* device_error_flag();

// Tensor map of an activation of type KDA_IO_* (no swizzle; a box reads zeros outside the tensor): `rank` dims and box
// sides, innermost first, and the byte strides of all but the innermost.  False where the driver takes no such map.
// Defined in kda_api.cu.
bool encode_tiled_map(void* map, const void* base, int dtype, int rank, const unsigned long long* dims,
                     const unsigned long long* strides, const unsigned* box);

}  // namespace kda
