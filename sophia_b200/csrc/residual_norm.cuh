// What stands between two mixers of a stack, per row of D channels:
//   u = o or rms_norm(o) w_b               (the branch, normed behind its block)
//   u = u sigmoid(g), u = dropout(u)       (its gate, and dropout)
//   v = x + scale u                        (the residual stream)
//   n = rms_norm(v) w                      (what the next block reads)
// with rms_norm(a) = a / sqrt(mean(a^2) + eps), forward and backward, every tensor
// read and written once.  Backward, with r_b and r the reciprocal roots (kept),
// t = dn w and m = keep / (1 - p):
//   dw = sum dn v r,   dv' = dv + r (t - v r^2 mean(t v)),   dx = dv'
//   dscale = sum dv' m s u,   du = dv' scale m s,   dg = dv' scale m u s (1 - s)
//   dw_b = sum du o r_b,      do = r_b (du w_b - o r_b^2 mean(du w_b o))
// (s the gate's sigmoid, u the branch behind its norm).  The sums over rows go by
// CTA into partial rows, summed in order by one more kernel.
//
// HBM-bound: 10 bytes an element forward and 16 backward when all is 16-bit.  W
// warps own a row, K pieces of V channels a thread; the row stays in registers
// between its two reductions.
//
// Dropout draws 32 bits per element from Philox4x32-10 (Salmon, Moraes, Dror and Shaw,
// 2011): key = the seed, counter = (channel / 4, row, row >> 32, offset), the four words
// for four neighbouring channels; an element is dropped where its word is below p 2^32.
// The backward draws the same words again; no mask is stored.
#pragma once

#include "ssm_common.cuh"

namespace kda {

constexpr int RN_MAX_WARPS = 16;
constexpr int RN_MAX_WIDTH = 8192;

struct RnParams {
  RowView x, o, g, dv, dn;  // g.p null = no gate; backward: dv.p / dn.p null = no gradient of that output
  const float *w, *wb, *scale;  // null = no next norm, no branch norm, no scale
  const long long* seed_ptr;    // device, or null: `seed`
  unsigned long long seed;
  unsigned offset, drop;  // an element is dropped where its word is below `drop`; drop_all: p = 1
  float keep_scale;
  bool dropout, drop_all;
  void *v, *n, *dx, *d_o, *dg;
  float* rstd;     // [rows][2]: r_b, r
  float* partial;  // [gridDim.x][3][D]: dw, dw_b, dscale
  long long rows;
  int T;  // rows per batch entry, or 0 where all rows of every tensor have one stride (no division)
  int D, warps;
  float eps;
};

// ---------------------------------------------------------------- rows

// V channels in pieces of up to 16 bytes.
template <typename T, int V>
struct RnVec {
  static constexpr int PER = V * sizeof(T) > 16 ? 16 / (int)sizeof(T) : V;
  IoVec<T, PER> p[V / PER];
  __device__ __forceinline__ void load(const T* q) {
#pragma unroll
    for (int i = 0; i < V / PER; ++i) p[i] = reinterpret_cast<const IoVec<T, PER>*>(q)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V / PER; ++i)
#pragma unroll
      for (int j = 0; j < PER; ++j) p[i].v[j] = io_from_f<T>(0.f);
  }
  __device__ __forceinline__ float get(int i) const { return io_to_f(p[i / PER].v[i % PER]); }
};
template <typename T, int V>
__device__ __forceinline__ void rn_store(T* q, const float (&f)[V]) {
  constexpr int PER = RnVec<T, V>::PER;
#pragma unroll
  for (int i = 0; i < V / PER; ++i) {
    IoVec<T, PER> r;
#pragma unroll
    for (int j = 0; j < PER; ++j) r.v[j] = io_from_f<T>(f[i * PER + j]);
    reinterpret_cast<IoVec<T, PER>*>(q)[i] = r;
  }
}
template <int V>
__device__ __forceinline__ void rn_param(const float* p, int c, float (&f)[V]) {
  constexpr int PER = V > 4 ? 4 : V;
#pragma unroll
  for (int i = 0; i < V / PER; ++i) {
    const IoVec<float, PER> r = reinterpret_cast<const IoVec<float, PER>*>(p + c)[i];
#pragma unroll
    for (int j = 0; j < PER; ++j) f[i * PER + j] = r.v[j];
  }
}
template <typename T>
__device__ __forceinline__ const T* rn_row(const RowView& r, long long row, int T_) {
  if (T_ == 0) return static_cast<const T*>(r.p) + row * r.st;
  const long long b = row / T_;
  return static_cast<const T*>(r.p) + b * r.sb + (row - b * T_) * r.st;
}

// Sum over the `warps` warps of a row's group, the same in every thread.  `slot` alternates, so that one barrier is enough.
__device__ __forceinline__ float rn_sum(float a, float (*part)[RN_MAX_WARPS], int slot, int group, int warps) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) a += __shfl_xor_sync(0xffffffffu, a, m);
  if (warps == 1) return a;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) part[slot][warp] = a;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
  float t = 0.f;
  for (int w = 0; w < warps; ++w) t += part[slot][group * warps + w];
  return t;
}

// ---------------------------------------------------------------- dropout

__device__ __forceinline__ uint4 philox(uint4 c, unsigned k0, unsigned k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const unsigned h0 = __umulhi(0xD2511F53u, c.x), l0 = 0xD2511F53u * c.x;
    const unsigned h1 = __umulhi(0xCD9E8D57u, c.z), l1 = 0xCD9E8D57u * c.z;
    c = make_uint4(h1 ^ c.y ^ k0, l1, h0 ^ c.w ^ k1, l0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}
// keep / (1 - p) of the V channels from c on (V = 1, or a multiple of 4 with c a multiple of 4)
template <int V>
__device__ __forceinline__ void rn_keep(const RnParams& P, unsigned k0, unsigned k1, long long row, int c, float (&m)[V]) {
  if (!P.dropout) {
#pragma unroll
    for (int i = 0; i < V; ++i) m[i] = 1.f;
    return;
  }
#pragma unroll
  for (int q = 0; q < (V + 3) / 4; ++q) {
    const uint4 r = philox(make_uint4((unsigned)c / 4 + q, (unsigned)row, (unsigned)(row >> 32), P.offset), k0, k1);
    const unsigned word[4] = {r.x, r.y, r.z, r.w};
    if (V == 1) {
      const unsigned w = (c & 2) ? ((c & 1) ? r.w : r.z) : ((c & 1) ? r.y : r.x);
      m[0] = w < P.drop || P.drop_all ? 0.f : P.keep_scale;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (q * 4 + i < V) m[q * 4 + i] = word[i] < P.drop || P.drop_all ? 0.f : P.keep_scale;
    }
  }
}
// a product with keep / (1 - p) that is 0 where the element is dropped, whatever it holds
__device__ __forceinline__ float rn_drop(float m, float a) { return m == 0.f ? 0.f : m * a; }

// ---------------------------------------------------------------- forward

template <typename TX, typename TO, int V, int K>
__global__ void __launch_bounds__(512) rn_fwd_kernel(const __grid_constant__ RnParams P) {
  __shared__ float part[2][RN_MAX_WARPS];
  const int warps = P.warps, group = (threadIdx.x >> 5) / warps, groups = (blockDim.x >> 5) / warps;
  const int me = threadIdx.x - group * warps * 32, stride = warps * 32 * V;
  const unsigned long long seed = P.seed_ptr ? (unsigned long long)*P.seed_ptr : P.seed;
  const unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  const float inv = 1.f / P.D;
  for (long long row = (long long)blockIdx.x * groups + group; row < P.rows; row += (long long)gridDim.x * groups) {
    const TX* px = rn_row<TX>(P.x, row, P.T);
    const TO* po = rn_row<TO>(P.o, row, P.T);
    const TO* pg = P.g.p ? rn_row<TO>(P.g, row, P.T) : nullptr;
    RnVec<TO, V> o[K], g[K];
    RnVec<TX, V> x[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = me * V + k * stride;
      if (c < P.D) {
        o[k].load(po + c);
        x[k].load(px + c);
        if (pg) g[k].load(pg + c);
      } else {
        o[k].zero();
        x[k].zero();
      }
    }
    float rb = 1.f;
    if (P.wb) {
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) ss = fmaf(o[k].get(i), o[k].get(i), ss);
      rb = rsqrtf(fmaf(rn_sum(ss, part, 0, group, warps), inv, P.eps));
    }
    float v[K][V], ss = 0.f;
    TX* pv = static_cast<TX*>(P.v) + row * P.D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = me * V + k * stride;
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = 0.f;
      if (c < P.D) {
        float f[V], m[V], u[V];
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = o[k].get(i);
        if (P.wb) {
          rn_param<V>(P.wb, c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) u[i] *= rb * f[i];
        }
        if (pg)
#pragma unroll
          for (int i = 0; i < V; ++i) u[i] *= sigmoidf_(g[k].get(i));
        if (P.dropout) {
          rn_keep<V>(P, k0, k1, row, c, m);
#pragma unroll
          for (int i = 0; i < V; ++i) u[i] = rn_drop(m[i], u[i]);
        }
        if (P.scale) {
          rn_param<V>(P.scale, c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) u[i] *= f[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[k][i] = x[k].get(i) + u[i];
          ss = fmaf(v[k][i], v[k][i], ss);
        }
        rn_store<TX, V>(pv + c, v[k]);
      }
    }
    float r = 0.f;
    if (P.w) {
      r = rsqrtf(fmaf(rn_sum(ss, part, 1, group, warps), inv, P.eps));
      TO* pn = static_cast<TO*>(P.n) + row * P.D;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = me * V + k * stride;
        if (c < P.D) {
          float f[V];
          rn_param<V>(P.w, c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] *= v[k][i] * r;
          rn_store<TO, V>(pn + c, f);
        }
      }
    }
    if (P.rstd && me == 0) {
      P.rstd[2 * row] = rb;
      P.rstd[2 * row + 1] = r;
    }
    if (warps > 1 && !(P.wb && P.w))  // one reduction a row: its slot is written again for the next row
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
  }
}

// ---------------------------------------------------------------- backward

template <typename TX, typename TO, int V, int K>
__global__ void __launch_bounds__(512) rn_bwd_kernel(const __grid_constant__ RnParams P) {
  extern __shared__ __align__(16) float acc[];  // [groups][3][D]: every thread adds to its own channels
  __shared__ float part[2][RN_MAX_WARPS];
  const int warps = P.warps, group = (threadIdx.x >> 5) / warps, groups = (blockDim.x >> 5) / warps;
  const int me = threadIdx.x - group * warps * 32, stride = warps * 32 * V;
  const unsigned long long seed = P.seed_ptr ? (unsigned long long)*P.seed_ptr : P.seed;
  const unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  const float inv = 1.f / P.D;
  float* sums = acc + (long long)group * 3 * P.D;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = me * V + k * stride;
    if (c < P.D)
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int i = 0; i < V; ++i) sums[q * P.D + c + i] = 0.f;
  }
  auto add = [&](int q, int c, const float (&f)[V]) {
    constexpr int PER = V > 4 ? 4 : V;
    IoVec<float, PER>* s = reinterpret_cast<IoVec<float, PER>*>(sums + q * P.D + c);
#pragma unroll
    for (int i = 0; i < V / PER; ++i) {
      IoVec<float, PER> t = s[i];
#pragma unroll
      for (int j = 0; j < PER; ++j) t.v[j] += f[i * PER + j];
      s[i] = t;
    }
  };
  for (long long row = (long long)blockIdx.x * groups + group; row < P.rows; row += (long long)gridDim.x * groups) {
    const TX* px = rn_row<TX>(P.x, row, P.T);
    const TO* po = rn_row<TO>(P.o, row, P.T);
    const TO* pg = P.g.p ? rn_row<TO>(P.g, row, P.T) : nullptr;
    const TX* pdv = P.dv.p ? rn_row<TX>(P.dv, row, P.T) : nullptr;
    const TO* pdn = P.dn.p ? rn_row<TO>(P.dn, row, P.T) : nullptr;
    RnVec<TO, V> o[K], g[K], dn[K];
    RnVec<TX, V> x[K], dv[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = me * V + k * stride;
      o[k].zero(), g[k].zero(), dn[k].zero(), x[k].zero(), dv[k].zero();
      if (c < P.D) {
        o[k].load(po + c);
        x[k].load(px + c);
        if (pg) g[k].load(pg + c);
        if (pdv) dv[k].load(pdv + c);
        if (pdn) dn[k].load(pdn + c);
      }
    }
    const float rb = P.rstd[2 * row], r = P.rstd[2 * row + 1];
    // the stream again, and the next norm's mean(t v)
    float v[K][V], m[K][V], dot = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = me * V + k * stride;
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = 0.f, m[k][i] = 0.f;
      if (c < P.D) {
        float f[V], u[V];
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = o[k].get(i);
        if (P.wb) {
          rn_param<V>(P.wb, c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) u[i] *= rb * f[i];
        }
        if (pg)
#pragma unroll
          for (int i = 0; i < V; ++i) u[i] *= sigmoidf_(g[k].get(i));
        rn_keep<V>(P, k0, k1, row, c, m[k]);
        if (P.scale) rn_param<V>(P.scale, c, f);
#pragma unroll
        for (int i = 0; i < V; ++i) v[k][i] = x[k].get(i) + rn_drop(m[k][i], u[i]) * (P.scale ? f[i] : 1.f);
        if (pdn) {
          rn_param<V>(P.w, c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) dot = fmaf(f[i] * dn[k].get(i), v[k][i], dot);
        }
      }
    }
    float mean = 0.f;
    if (pdn) mean = rn_sum(dot, part, 0, group, warps) * inv * r * r;
    dot = 0.f;
    float du[K][V];
    TX* pdx = static_cast<TX*>(P.dx) + row * P.D;
    TO* pdg = static_cast<TO*>(P.dg) + row * P.D;
    TO* pdo = static_cast<TO*>(P.d_o) + row * P.D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = me * V + k * stride;
#pragma unroll
      for (int i = 0; i < V; ++i) du[k][i] = 0.f;
      if (c < P.D) {
        float d[V], f[V], t[V], wb[V];
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = dv[k].get(i);
        if (pdn) {
          rn_param<V>(P.w, c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            d[i] = fmaf(r, fmaf(-v[k][i], mean, f[i] * dn[k].get(i)), d[i]);
            t[i] = dn[k].get(i) * v[k][i] * r;
          }
          add(0, c, t);
        }
        rn_store<TX, V>(pdx + c, d);
        if (P.wb) rn_param<V>(P.wb, c, wb);
        if (P.scale) rn_param<V>(P.scale, c, f);
        float u[V], s[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          u[i] = P.wb ? o[k].get(i) * rb * wb[i] : o[k].get(i);
          s[i] = pg ? sigmoidf_(g[k].get(i)) : 1.f;
          const float dm = rn_drop(m[k][i], d[i]);           // gradient of scale u s
          t[i] = m[k][i] == 0.f ? 0.f : dm * (u[i] * s[i]);  // of scale
          const float ds = P.scale ? dm * f[i] : dm;         // of u s
          du[k][i] = m[k][i] == 0.f ? 0.f : ds * s[i];
          s[i] = m[k][i] == 0.f ? 0.f : ds * u[i] * (s[i] * (1.f - s[i]));
        }
        if (P.scale) add(2, c, t);
        if (pg) rn_store<TO, V>(pdg + c, s);
        if (P.wb) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            t[i] = du[k][i] * o[k].get(i) * rb;
            du[k][i] *= wb[i];
            dot = fmaf(du[k][i], o[k].get(i), dot);
          }
          add(1, c, t);
        } else {
          rn_store<TO, V>(pdo + c, du[k]);
        }
      }
    }
    if (P.wb) {
      mean = rn_sum(dot, part, 1, group, warps) * inv * rb * rb;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = me * V + k * stride;
        if (c < P.D) {
#pragma unroll
          for (int i = 0; i < V; ++i) du[k][i] = rb * fmaf(-o[k].get(i), mean, du[k][i]);
          rn_store<TO, V>(pdo + c, du[k]);
        }
      }
    }
    if (warps > 1 && !(P.wb && pdn)) asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 3 * P.D; i += blockDim.x) {  // the CTA's sums, its groups in order
    float t = 0.f;
    for (int q = 0; q < groups; ++q) t += acc[(long long)q * 3 * P.D + i];
    P.partial[(long long)blockIdx.x * 3 * P.D + i] = t;
  }
}

// The sums over the CTAs' partial rows [parts][3][D]: eight strided slices of the rows in order, then the slices
// in order.  Outputs may be null.
constexpr int RN_REDUCE_COLS = 32, RN_REDUCE_SLICES = 8;
static __global__ void __launch_bounds__(RN_REDUCE_COLS * RN_REDUCE_SLICES)
    rn_reduce_kernel(const float* partial, int parts, int D, float* dw, float* dwb, float* dscale) {
  __shared__ float part[RN_REDUCE_SLICES][RN_REDUCE_COLS];
  const int c = threadIdx.x % RN_REDUCE_COLS, sl = threadIdx.x / RN_REDUCE_COLS;
  const int k = blockIdx.x * RN_REDUCE_COLS + c;
  float* out = blockIdx.y == 0 ? dw : (blockIdx.y == 1 ? dwb : dscale);
  if (!out) return;
  float acc = 0.f;
  if (k < D)
#pragma unroll 8
    for (int b = sl; b < parts; b += RN_REDUCE_SLICES) acc += partial[((long long)b * 3 + blockIdx.y) * D + k];
  part[sl][c] = acc;
  __syncthreads();
  if (sl != 0 || k >= D) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < RN_REDUCE_SLICES; ++i) t += part[i][c];
  out[k] = t;
}

}  // namespace kda
