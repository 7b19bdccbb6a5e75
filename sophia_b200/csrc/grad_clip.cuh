// Global gradient norm over many tensors, and clipping:
//   norm = sqrt(sum over all elements of g^2),
//   out  = g * min(1, max_norm / (norm + eps)).
//
// Memory bound: the gradients are read once for the norm and once more for the
// scaling, which writes the output; a sum below the L2's size finds its second
// read there, so the scaling walks the chunks backwards.  The tensors' addresses travel
// as a kernel parameter (no copy, no host wait); each launch takes up to
// GRAD_MAX_TENSORS of them.  A CTA takes a run of chunks of GRAD_CHUNK elements.  Squares
// are summed in fp32 over at most GRAD_CHUNK / GRAD_THREADS elements of a thread
// and in fp64 from there on, in an order that depends on the sizes, on the addresses modulo 16
// bytes and on the number of SMs, never on timing.  Where fp32 squares would overflow or vanish the thread sums its
// elements again in fp64, so the norm is right over the whole range of fp32.
// Measured, 455 M elements of bf16 in 336 tensors to fp32: norm 152 us (6.0 TB/s), scaling
// 487 us (5.6 TB/s); chunks of 4096 elements 178 and 479 us, of 8192 157 and 486 us.
#pragma once

#include "ssm_common.cuh"

namespace kda {

constexpr int GRAD_THREADS = 256;
constexpr int GRAD_CHUNK = 16384;
constexpr int GRAD_MAX_TENSORS = 1024;  // 30 KB of kernel parameters
constexpr int GRAD_FEW_TENSORS = 64;    // the smaller table: 2 KB

template <int M>
struct GradTable {
  const void* in[M];
  void* out[M];
  long long numel[M];
  int chunk0[M + 1];  // chunks before tensor i
  unsigned char tin[M], tout[M];  // 0 fp32, 1 bf16, 2 fp16
  int n;
};

// The chunks of a CTA: a run of neighbours, so that the tensor of the next one is found by
// walking on from the last (its table entry stays in registers meanwhile).
template <int M>
struct GradWalk {
  int first, end;  // chunks of this CTA
  int i;           // tensor of the current chunk
  __device__ __forceinline__ explicit GradWalk(const GradTable<M>& tab) {
    const int chunks = tab.chunk0[tab.n], per = (chunks + gridDim.x - 1) / gridDim.x;
    first = min((int)blockIdx.x * per, chunks);
    end = min(first + per, chunks);
    int lo = 0, hi = tab.n;
    while (hi - lo > 1) {  // the last tensor that starts at or before the first chunk
      const int mid = (lo + hi) >> 1;
      if (tab.chunk0[mid] <= first) lo = mid; else hi = mid;
    }
    i = lo;
  }
  __device__ __forceinline__ void to(const GradTable<M>& tab, int chunk) {
    while (tab.chunk0[i + 1] <= chunk) ++i;
    while (tab.chunk0[i] > chunk) --i;
  }
};

// A thread's share of a chunk in pieces, fn(piece): 16 bytes each when the address allows, else elements.
template <typename T, typename F>
__device__ __forceinline__ void grad_each(const T* p, int n, F fn) {
  constexpr int V = 16 / sizeof(T), U = 4;
  int k = threadIdx.x;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const IoVec<T, V>* q = reinterpret_cast<const IoVec<T, V>*>(p);
    const int nv = n / V;
    int i = threadIdx.x;
    for (; i + (U - 1) * GRAD_THREADS < nv; i += U * GRAD_THREADS) {
      IoVec<T, V> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = q[i + u * GRAD_THREADS];
#pragma unroll
      for (int u = 0; u < U; ++u) fn(r[u]);
    }
    for (; i < nv; i += GRAD_THREADS) fn(q[i]);
    k += nv * V;
  }
  for (; k < n; k += GRAD_THREADS) fn(*reinterpret_cast<const IoVec<T, 1>*>(p + k));
}
// The bits of a piece's elements, joined: zero where all of them are (signs stay in).
template <typename T, int V>
__device__ __forceinline__ uint32_t grad_bits(const IoVec<T, V>& r) {
  if (sizeof(T) * V < 4) return *reinterpret_cast<const unsigned short*>(&r);
  uint32_t b = 0;
#pragma unroll
  for (int w = 0; w < (int)sizeof(T) * V / 4; ++w) b |= reinterpret_cast<const uint32_t*>(&r)[w];
  return b;
}

// Sum of squares of a thread's elements: in fp32, and again in fp64 where fp32 squares leave their range -- the
// sum is not finite (one element above 1.8e19 is enough), or so small that squares below 2^-126 may have lost
// their digits in it (64 of them, each off by 2^-150, are 2^-44 of a sum of 2^-100).  `bits` tells small elements from
// zeros.
template <typename T>
__device__ __forceinline__ double grad_sumsq(const T* p, int n) {
  float acc = 0.f;
  uint32_t bits = 0;
  grad_each(p, n, [&](const auto& r) {
#pragma unroll
    for (const T v : r.v) {
      const float f = io_to_f(v);
      acc = fmaf(f, f, acc);
    }
    bits |= grad_bits(r);
  });
  if (acc >= 0x1p-100f && acc < INFINITY) return acc;
  if ((bits & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)) == 0) return 0;
  double wide = 0;
  grad_each(p, n, [&](const auto& r) {
    for (const T v : r.v) {
      const double f = io_to_f(v);
      wide = fma(f, f, wide);
    }
  });
  return wide;
}

// Sum over the CTA in a fixed order; valid in thread 0.
__device__ __forceinline__ double grad_block_sum(double v) {
  __shared__ double red[GRAD_THREADS / 32];
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0;
  if (threadIdx.x == 0)
    for (int i = 0; i < GRAD_THREADS / 32; ++i) t += red[i];
  __syncthreads();
  return t;
}

template <int M>
__global__ void __launch_bounds__(GRAD_THREADS) grad_norm_kernel(const __grid_constant__ GradTable<M> tab,
                                                                 double* partial) {
  GradWalk<M> walk(tab);
  double acc = 0;
  for (int ch = walk.first; ch < walk.end; ++ch) {
    walk.to(tab, ch);
    const int i = walk.i;
    const long long at = (long long)(ch - tab.chunk0[i]) * GRAD_CHUNK;
    const int n = (int)min((long long)GRAD_CHUNK, tab.numel[i] - at);
    double s;
    if (tab.tin[i] == 0) s = grad_sumsq(static_cast<const float*>(tab.in[i]) + at, n);
    else if (tab.tin[i] == 1) s = grad_sumsq(static_cast<const bf16*>(tab.in[i]) + at, n);
    else s = grad_sumsq(static_cast<const f16*>(tab.in[i]) + at, n);
    acc += s;
  }
  acc = grad_block_sum(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// Pieces that take 16 bytes on the wider side, four in flight per thread, when both addresses
// allow.
template <typename TI, typename TO>
__device__ __forceinline__ void grad_scale(const TI* p, TO* q, int n, float coef) {
  constexpr int V = 16 / (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO)), U = 4;
  if (((reinterpret_cast<uintptr_t>(p) & (V * sizeof(TI) - 1)) | (reinterpret_cast<uintptr_t>(q) & (V * sizeof(TO) - 1))) ==
      0) {
    const int nv = n / V;
    int i = threadIdx.x;
    for (; i + (U - 1) * GRAD_THREADS < nv; i += U * GRAD_THREADS) {
      float f[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) io_load<TI, V>(p + (i + u * GRAD_THREADS) * V, f[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int k = 0; k < V; ++k) f[u][k] *= coef;
        io_store<TO, V>(q + (i + u * GRAD_THREADS) * V, f[u]);
      }
    }
    for (; i < nv; i += GRAD_THREADS) {
      float f[V];
      io_load<TI, V>(p + i * V, f);
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] *= coef;
      io_store<TO, V>(q + i * V, f);
    }
    for (int k = nv * V + threadIdx.x; k < n; k += GRAD_THREADS) q[k] = io_from_f<TO>(io_to_f(p[k]) * coef);
  } else {
    for (int k = threadIdx.x; k < n; k += GRAD_THREADS) q[k] = io_from_f<TO>(io_to_f(p[k]) * coef);
  }
}

template <typename TI>
__device__ __forceinline__ void grad_scale_to(const TI* p, void* q, long long at, int n, float coef, int tout) {
  if (tout == 0) grad_scale(p, static_cast<float*>(q) + at, n, coef);
  else if (tout == 1) grad_scale(p, static_cast<bf16*>(q) + at, n, coef);
  else grad_scale(p, static_cast<f16*>(q) + at, n, coef);
}

// Every CTA sums the same `parts` partials in the same order.
__device__ __forceinline__ double grad_total(const double* partial, int parts) {
  double v = 0;
  for (int i = threadIdx.x; i < parts; i += GRAD_THREADS) v += partial[i];
  return grad_block_sum(v);
}

// norm = sqrt(sum of partials), alone.
__global__ void __launch_bounds__(GRAD_THREADS) grad_norm_finish_kernel(const double* partial, int parts, float* norm) {
  const double t = grad_total(partial, parts);
  if (threadIdx.x == 0) *norm = (float)sqrt(t);
}

template <int M>
__global__ void __launch_bounds__(GRAD_THREADS) grad_scale_kernel(const __grid_constant__ GradTable<M> tab,
                                                                  const double* partial, int parts, float max_norm,
                                                                  float eps, float* norm) {
  __shared__ float s_coef;
  const double t = grad_total(partial, parts);
  if (threadIdx.x == 0) {
    const float nrm = (float)sqrt(t);
    const float c = max_norm / (nrm + eps);
    s_coef = c > 1.f ? 1.f : c;  // a NaN norm stays NaN
    if (blockIdx.x == 0 && norm) *norm = nrm;
  }
  __syncthreads();
  const float coef = s_coef;
  GradWalk<M> walk(tab);
  for (int ch = walk.end - 1; ch >= walk.first; --ch) {
    walk.to(tab, ch);
    const int i = walk.i;
    if (coef == 1.f && tab.in[i] == tab.out[i]) continue;  // a product by one, in place
    const long long at = (long long)(ch - tab.chunk0[i]) * GRAD_CHUNK;
    const int n = (int)min((long long)GRAD_CHUNK, tab.numel[i] - at);
    if (tab.tin[i] == 0) grad_scale_to(static_cast<const float*>(tab.in[i]) + at, tab.out[i], at, n, coef, tab.tout[i]);
    else if (tab.tin[i] == 1)
      grad_scale_to(static_cast<const bf16*>(tab.in[i]) + at, tab.out[i], at, n, coef, tab.tout[i]);
    else
      grad_scale_to(static_cast<const f16*>(tab.in[i]) + at, tab.out[i], at, n, coef, tab.tout[i]);
  }
}

}  // namespace kda
