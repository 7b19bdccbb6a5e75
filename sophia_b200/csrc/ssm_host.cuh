// Host-side helpers of the entry points whose activations are strided rows
// [B, T, width]: argument checks, packed-sequence maps, states handed through.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <string>

#include "kda_host.h"
#include "ssm_common.cuh"

namespace kda {

inline size_t io_size(int dtype) { return dtype == KDA_IO_F32 ? 4 : 2; }

inline int check_dtype(int dtype) {
  if (dtype < KDA_IO_F32 || dtype > KDA_IO_F16)
    return fail(KDA_ERR_INVALID, "dtype must be KDA_IO_F32, KDA_IO_BF16 or KDA_IO_F16");
  return KDA_OK;
}

// Sequences of a call: B rows of T tokens, or (cu) one row of N packed ones.
inline int check_rows(long long B, long long T, int N, const int32_t* cu) {
  if (B < 1 || T < 0 || N < 1) return fail(KDA_ERR_INVALID, "B >= 1, T >= 0 and N >= 1 are required");
  if (cu && B != 1)
    return fail(KDA_ERR_INVALID, "The batch size is expected to be 1 rather than " + std::to_string(B) +
                                     " when using `cu_seqlens`.");
  if (!cu && N != B) return fail(KDA_ERR_INVALID, "N must equal B without cu_seqlens");
  if (B > 65535) return fail(KDA_ERR_UNSUPPORTED, "more than 65535 rows");
  if (T > INT32_MAX / 2) return fail(KDA_ERR_UNSUPPORTED, "too many tokens");
  return KDA_OK;
}

inline bool vec_rows(const void* p, long long sb, long long st, long long B, long long T, int elems, size_t esz) {
  return aligned(p, (size_t)elems * esz) && (B <= 1 || sb % elems == 0) && (T <= 1 || st % elems == 0);
}

inline size_t map_bytes(long long T, bool packed) { return packed ? 2 * align256((size_t)std::max(T, 1LL) * 4) : 0; }

// Sequence maps of a packed call, and the rows of empty sequences (dst <- src).
inline int build_map(SeqMap& m, Carver& cv, const int32_t* cu, int T, int N, const float* src, float* dst, long long per,
              cudaStream_t st) {
  m.start = m.end = nullptr;
  m.T = T;
  if (!cu) return KDA_OK;
  int* err = device_error_flag();
  if (!err) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  int* start = cv.take<int>((size_t)T * 4);
  int* end = cv.take<int>((size_t)T * 4);
  SeqMapParams p{cu, N, T, start, end, src, dst, per, err};
  const int blocks = (T + SEQ_MAP_THREADS - 1) / SEQ_MAP_THREADS + std::min(N, 2 * sm_count());
  {
    TimedLaunch tl(K_TABLE, st);
    ssm_seq_map_kernel<<<blocks, SEQ_MAP_THREADS, 0, st>>>(p);
  }
  m.start = start;
  m.end = end;
  return launch_check("sequence map");
}

// T = 0: every sequence is empty, its state goes through.
inline int pass_state(const float* src, float* dst, long long elems, cudaStream_t st) {
  if (!dst || elems == 0) return KDA_OK;
  const cudaError_t e = src ? cudaMemcpyAsync(dst, src, (size_t)elems * 4, cudaMemcpyDeviceToDevice, st)
                            : cudaMemsetAsync(dst, 0, (size_t)elems * 4, st);
  return e == cudaSuccess ? KDA_OK : fail(KDA_ERR_CUDA, cudaGetErrorString(e));
}
inline int zero_floats(float* p, long long elems, cudaStream_t st) { return pass_state(nullptr, p, elems, st); }

}  // namespace kda

#define SSM_DISPATCH(dtype, fn, ...)                              \
  ((dtype) == KDA_IO_F32    ? fn<float>(__VA_ARGS__)              \
   : (dtype) == KDA_IO_BF16 ? fn<bf16>(__VA_ARGS__)               \
                            : fn<f16>(__VA_ARGS__))
