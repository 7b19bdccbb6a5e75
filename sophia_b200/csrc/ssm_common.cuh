// Shared device helpers of the state-space operators (short_conv,
// selective_scan and their single-token steps).
//
// Activations are fp32, bf16 or fp16 rows [B, T, width] whose last dimension is
// contiguous; batch and token strides are free (a slice of a wider projection
// is read in place).  Arithmetic, states and sums are fp32; a value is rounded
// to the activations' type once, when it is stored.
#pragma once

#include <cuda_fp16.h>

#include "kda_common.cuh"

namespace kda {

typedef __half f16;

__device__ __forceinline__ float io_to_f(float v) { return v; }
__device__ __forceinline__ float io_to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float io_to_f(f16 v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T io_from_f(float v);
template <> __device__ __forceinline__ float io_from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 io_from_f<bf16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ f16 io_from_f<f16>(float v) { return __float2half(v); }

// V consecutive elements as one load or store of V * sizeof(T) bytes (the
// address is a multiple of that).
template <typename T, int V> struct alignas(sizeof(T) * V) IoVec { T v[V]; };
template <typename T, int V>
__device__ __forceinline__ void io_load(const T* p, float (&f)[V]) {
  const IoVec<T, V> r = *reinterpret_cast<const IoVec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = io_to_f(r.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void io_store(T* p, const float (&f)[V]) {
  IoVec<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = io_from_f<T>(f[i]);
  *reinterpret_cast<IoVec<T, V>*>(p) = r;
}

// S values of one kind that a thread owns, pairs in packed fp32 arithmetic.
typedef unsigned long long u64;
__device__ __forceinline__ u64 pk2(float lo, float hi) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 upk2(u64 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <int S>
struct Lane {
  static_assert(S % 2 == 0, "pairs");
  u64 p[S / 2];
  __device__ __forceinline__ float get(int i) const { return i & 1 ? upk2(p[i / 2]).y : upk2(p[i / 2]).x; }
  __device__ __forceinline__ void set(int i, float v) {
    const float2 o = upk2(p[i / 2]);
    p[i / 2] = i & 1 ? pk2(o.x, v) : pk2(v, o.y);
  }
  __device__ __forceinline__ static Lane of(const float (&f)[S]) {
    Lane r;
#pragma unroll
    for (int k = 0; k < S / 2; ++k) r.p[k] = pk2(f[2 * k], f[2 * k + 1]);
    return r;
  }
  __device__ __forceinline__ static Lane load(const float* q) {  // S * 4 bytes, aligned
    Lane r;
    if (S % 4 == 0) {
#pragma unroll
      for (int k = 0; k < S / 4; ++k) {
        const ulonglong2 v = reinterpret_cast<const ulonglong2*>(q)[k];
        r.p[2 * k] = v.x;
        r.p[2 * k + 1] = v.y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < S / 2; ++k) r.p[k] = reinterpret_cast<const u64*>(q)[k];
    }
    return r;
  }
  __device__ __forceinline__ void store(float* q) const {
    if (S % 4 == 0) {
#pragma unroll
      for (int k = 0; k < S / 4; ++k) reinterpret_cast<ulonglong2*>(q)[k] = make_ulonglong2(p[2 * k], p[2 * k + 1]);
    } else {
#pragma unroll
      for (int k = 0; k < S / 2; ++k) reinterpret_cast<u64*>(q)[k] = p[k];
    }
  }
  __device__ __forceinline__ static Lane all(float v) {
    Lane r;
#pragma unroll
    for (int k = 0; k < S / 2; ++k) r.p[k] = pk2(v, v);
    return r;
  }
  __device__ __forceinline__ Lane exp2() const {
    Lane r;
#pragma unroll
    for (int k = 0; k < S / 2; ++k) {
      const float2 f = upk2(p[k]);
      r.p[k] = pk2(ex2(f.x), ex2(f.y));
    }
    return r;
  }
  friend __device__ __forceinline__ Lane operator*(const Lane& a, const Lane& b) {
    Lane r;
#pragma unroll
    for (int k = 0; k < S / 2; ++k) r.p[k] = mul2(a.p[k], b.p[k]);
    return r;
  }
  friend __device__ __forceinline__ Lane operator+(const Lane& a, const Lane& b) {
    Lane r;
#pragma unroll
    for (int k = 0; k < S / 2; ++k) r.p[k] = add2(a.p[k], b.p[k]);
    return r;
  }
  friend __device__ __forceinline__ Lane fma(const Lane& a, const Lane& b, const Lane& c) {
    Lane r;
#pragma unroll
    for (int k = 0; k < S / 2; ++k) r.p[k] = fma2(a.p[k], b.p[k], c.p[k]);
    return r;
  }
};
template <>
struct Lane<1> {
  float f;
  __device__ __forceinline__ float get(int) const { return f; }
  __device__ __forceinline__ void set(int, float v) { f = v; }
  __device__ __forceinline__ static Lane all(float v) { return {v}; }
  __device__ __forceinline__ Lane exp2() const { return {ex2(f)}; }
  friend __device__ __forceinline__ Lane operator*(const Lane& a, const Lane& b) { return {a.f * b.f}; }
  friend __device__ __forceinline__ Lane operator+(const Lane& a, const Lane& b) { return {a.f + b.f}; }
  friend __device__ __forceinline__ Lane fma(const Lane& a, const Lane& b, const Lane& c) { return {fmaf(a.f, b.f, c.f)}; }
};
// sum of a b over a lane's states
template <int S>
__device__ __forceinline__ float lane_dot(const Lane<S>& a, const Lane<S>& b) {
  u64 t = mul2(a.p[0], b.p[0]);
#pragma unroll
  for (int k = 1; k < S / 2; ++k) t = fma2(a.p[k], b.p[k], t);
  const float2 f = upk2(t);
  return f.x + f.y;
}
template <int S>
__device__ __forceinline__ Lane<S> lane_sigmoid(const Lane<S>& v) {
  Lane<S> d = (v * Lane<S>::all(-LOG2E)).exp2() + Lane<S>::all(1.f);
#pragma unroll
  for (int i = 0; i < S; ++i) d.set(i, rcp(d.get(i)));
  return d;
}
template <typename T, int S>
__device__ __forceinline__ Lane<S> lane_from(const IoVec<T, S>& v) {
  Lane<S> r = Lane<S>::all(0.f);
#pragma unroll
  for (int i = 0; i < S; ++i) r.set(i, io_to_f(v.v[i]));
  return r;
}
template <typename T, int S>
__device__ __forceinline__ void lane_store(T* p, const Lane<S>& v) {
  float f[S];
#pragma unroll
  for (int i = 0; i < S; ++i) f[i] = v.get(i);
  io_store<T, S>(p, f);
}

// A strided activation: element (b, t, c) at p + b*sb + t*st + c.
struct RowView {
  const void* p;
  long long sb, st;
};
template <typename T>
__device__ __forceinline__ const T* row_ptr(const RowView& r, long long b, long long t) {
  return static_cast<const T*>(r.p) + b * r.sb + t * r.st;
}

// Where sequences start and end.  Without the maps row b is one sequence of T
// tokens; with them (packed, one row) start[t] / end[t] is the sequence whose
// first / last token is t, or -1.
struct SeqMap {
  const int *start, *end;
  int T;
};
__device__ __forceinline__ int seq_start_at(const SeqMap& m, int b, int t) {
  return m.start ? __ldg(m.start + t) : (t == 0 ? b : -1);
}
__device__ __forceinline__ int seq_end_at(const SeqMap& m, int b, int t) {
  return m.end ? __ldg(m.end + t) : (t == m.T - 1 ? b : -1);
}

// softplus(x) = max(x, 0) + log(1 + e), e = e^-|x|, with log(1 + e) = 2 atanh(s),
// s = e / (2 + e) in [0, 1/3]: atanh(s) / s is a polynomial in s^2 (a Chebyshev
// fit, relative error 8e-9), so the result keeps fp32 relative accuracy where e
// is tiny and 1 + e would lose it.
__device__ __forceinline__ float softplusf_(float x) {
  const float e = ex2(-fabsf(x) * LOG2E), s = e * rcp(2.f + e), v = s * s;
  float q = fmaf(0.140807271f, v, 0.139821723f);
  q = fmaf(q, v, 0.20012325f);
  q = fmaf(q, v, 0.333331615f);
  q = fmaf(q, v, 1.f);
  return fmaf(2.f * s, q, fmaxf(x, 0.f));
}
__device__ __forceinline__ float siluf_(float v) { return v * sigmoidf_(v); }

// The pool entry of a single-token call's row: negative for a padding row; an entry past the pool is
// reported (device error 11) and treated as one.
__device__ __forceinline__ int step_slot(const int* slots, int r, int pool, int* err) {
  const int s = slots ? __ldg(slots + r) : r;
  if (s >= pool) {
    atomicExch(err, 11);
    return -1;
  }
  return s;
}

constexpr int SEQ_MAP_THREADS = 256;
constexpr int SEQ_MAP_TABLE = 4096;

struct SeqMapParams {
  const int* cu;  // [nseq + 1]
  int nseq, T;
  int *start, *end;
  const float* src;  // per-sequence rows that an empty sequence hands through (null = zeros)
  float* dst;        // null = nothing to hand through
  long long per;     // elements of a row
  int* err;
};

// Packed sequences: the maps of first and last tokens, by a binary search of
// every token in cu_seqlens (the last sequence that starts at or before it; an
// empty sequence holds no token), and the states of empty sequences.  A table
// that does not start at 0, decreases or does not end at T sets the device
// error 3; the maps still hold only valid sequence numbers.
static __global__ void __launch_bounds__(SEQ_MAP_THREADS) ssm_seq_map_kernel(SeqMapParams P) {
  __shared__ int table[SEQ_MAP_TABLE];
  const int tok_blocks = (P.T + SEQ_MAP_THREADS - 1) / SEQ_MAP_THREADS;
  if ((int)blockIdx.x < tok_blocks) {
    const int t = blockIdx.x * SEQ_MAP_THREADS + threadIdx.x;
    const int* cu = P.cu;
    if (P.nseq < SEQ_MAP_TABLE) {  // one read of global memory in a row, not one per halving
      for (int i = threadIdx.x; i <= P.nseq; i += SEQ_MAP_THREADS) table[i] = __ldg(P.cu + i);
      __syncthreads();
      cu = table;
    }
    if (t >= P.T) return;
    int lo = 0, hi = P.nseq;  // the answer is in [lo, hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t) lo = mid; else hi = mid;
    }
    P.start[t] = cu[lo] == t ? lo : -1;
    P.end[t] = cu[lo + 1] == t + 1 ? lo : -1;
    return;
  }
  const int first = (int)blockIdx.x - tok_blocks, step = (int)gridDim.x - tok_blocks;
  for (int i = first; i < P.nseq; i += step) {
    const int a = __ldg(P.cu + i), b = __ldg(P.cu + i + 1);
    if (threadIdx.x == 0 && (a > b || (i == 0 && a != 0) || (i == P.nseq - 1 && b != P.T))) atomicExch(P.err, 3);
    if (P.dst && a >= b)
      for (long long k = threadIdx.x; k < P.per; k += SEQ_MAP_THREADS)
        P.dst[i * P.per + k] = P.src ? P.src[i * P.per + k] : 0.f;
  }
}

// Rows of new states to their pool entries (elements of V floats, `per` of them a row); padding rows and rows past the
// pool as in the single-token calls.
template <typename V>
static __global__ void __launch_bounds__(256) ssm_put_states_kernel(const V* src, const int* slots, int rows, long long per,
                                                                    int pool, V* dst, int* err) {
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    const int s = step_slot(slots, r, pool, err);
    if (s < 0) continue;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < per; i += (long long)gridDim.x * blockDim.x)
      dst[s * per + i] = src[r * per + i];
  }
}

// Sums `parts` rows of `cols` = q * w1 columns, w1 = w0 + 1 or w0 + 2: 8 strided slices
// of the rows in order, then the slices in order -- a fixed order for a given
// number of rows.  Columns r < w0 of item q go to out0[q * w0 + r], the next to
// out1[q], the one after it to out2[q] (null: dropped).
constexpr int SSM_REDUCE_COLS = 32, SSM_REDUCE_SLICES = 8;
static __global__ void __launch_bounds__(SSM_REDUCE_COLS * SSM_REDUCE_SLICES)
    ssm_reduce_kernel(const float* partial, long long parts, long long cols, int w0, int w1, float* out0, float* out1,
                      float* out2) {
  __shared__ float part[SSM_REDUCE_SLICES][SSM_REDUCE_COLS];
  const int c = threadIdx.x % SSM_REDUCE_COLS, sl = threadIdx.x / SSM_REDUCE_COLS;
  const long long k = (long long)blockIdx.x * SSM_REDUCE_COLS + c;
  float acc = 0.f;
  if (k < cols)
#pragma unroll 8
    for (long long b = sl; b < parts; b += SSM_REDUCE_SLICES) acc += partial[b * cols + k];
  part[sl][c] = acc;
  __syncthreads();
  if (sl != 0 || k >= cols) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < SSM_REDUCE_SLICES; ++i) t += part[i][c];
  const long long q = k / w1;
  const int r = (int)(k - q * w1);
  if (r < w0) out0[q * w0 + r] = t;
  else if (r == w0 && out1) out1[q] = t;
  else if (r > w0 && out2) out2[q] = t;
}

}  // namespace kda
