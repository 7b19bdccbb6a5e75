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
  int stages, batch;  // of the ring: stages, and how many times a group's rows a stage holds
  unsigned dense;     // bit per tensor (x, o, g, dv, dn): rows lie end to end
  int D, warps, lanes;  // a row's threads: warps of a group, or (one warp) that many lanes
  int parts;  // CTAs of the backward, set by its launch
  int* err;
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
    const u64 p0 = (u64)0xD2511F53u * c.x, p1 = (u64)0xCD9E8D57u * c.z;
    c = make_uint4((unsigned)(p1 >> 32) ^ c.y ^ k0, (unsigned)p1, (unsigned)(p0 >> 32) ^ c.w ^ k1, (unsigned)p0);
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

// ---------------------------------------------------------------- rows by bulk copies

// Aligned rows come into a ring of stages in shared memory by bulk copies, so that the next rows are on their way
// while one is worked on.  A group of W warps owns a row at a time (of narrow rows `lanes` lanes of a single warp, which
// has 32 / lanes rows at once), and a stage holds enough consecutive rows for copies of a few KB: rows that lie end to
// end are one copy (small copies cost the copy engine as much as large ones).  A thread has at most 16 channels, the same
// in every row, in packed fp32 arithmetic; parameters (forward) and sums over rows (backward) stay in its registers.
constexpr int RN_MAX_STAGES = 4;
constexpr int RN_MAX_GROUPS = 8;

__device__ __forceinline__ void rn_bar_init(uint64_t* bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void rn_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void rn_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ bool rn_wait(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 26); ++i) {
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(smem_u32(bar)), "r"(parity)
                 : "memory");
    if (done) return true;
  }
  return false;
}

// Where a thread stands.
struct RnPlace {
  int group, mine;   // its group of the CTA, its number in it
  int per, sub, me;  // rows that a group works on at once, which of them, and its number in that row
  int stride;        // channels between a thread's pieces
  long long step, first;  // rows between a group's stages, and its first
};
template <int V>
__device__ __forceinline__ RnPlace rn_place(const RnParams& P) {
  RnPlace a;
  const int groups = (int)(blockDim.x >> 5) / P.warps;
  a.group = (int)(threadIdx.x >> 5) / P.warps;
  a.mine = threadIdx.x - a.group * P.warps * 32;
  a.per = P.warps > 1 ? 1 : 32 / P.lanes;
  a.sub = P.warps > 1 ? 0 : a.mine / P.lanes;
  a.me = P.warps > 1 ? a.mine : a.mine % P.lanes;
  a.stride = (P.warps > 1 ? P.warps * 32 : P.lanes) * V;
  const long long rows = (long long)a.per * P.batch;
  a.step = (long long)gridDim.x * groups * rows;
  a.first = ((long long)blockIdx.x * groups + a.group) * rows;
  return a;
}

// n rows of a tensor from row0 on to `dst`; `dense`: they lie end to end.  (Called by the first warp of a group.)
template <typename T>
__device__ __forceinline__ void rn_fetch(char* dst, const RowView& r, bool dense, long long row0, int n, const RnParams& P,
                                         uint64_t* bar) {
  const int lane = threadIdx.x & 31;
  const uint32_t bytes = P.D * (uint32_t)sizeof(T);
  if (dense) {
    if (lane == 0) rn_bulk(dst, rn_row<T>(r, row0, P.T), n * bytes, bar);
  } else {
    for (int i = lane; i < n; i += 32) rn_bulk(dst + (size_t)i * bytes, rn_row<T>(r, row0 + i, P.T), bytes, bar);
  }
}
// The sum over a row's threads: `lanes` of a warp, or `warps` warps.
__device__ __forceinline__ float rn_total(float a, float (*part)[RN_MAX_WARPS], int slot, int group, const RnParams& P) {
  if (P.warps > 1) return rn_sum(a, part, slot, group, P.warps);
  for (int m = P.lanes >> 1; m >= 1; m >>= 1) a += __shfl_xor_sync(0xffffffffu, a, m);
  return a;
}

// V channels as pairs.
template <typename T, int V>
__device__ __forceinline__ void rn_get(const T* q, u64 (&f)[V / 2]) {
  RnVec<T, V> v;
  v.load(q);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) f[i] = pk2(v.get(2 * i), v.get(2 * i + 1));
}
template <typename T, int V>
__device__ __forceinline__ void rn_put(T* q, const u64 (&f)[V / 2]) {
  float o[V];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 t = upk2(f[i]);
    o[2 * i] = t.x;
    o[2 * i + 1] = t.y;
  }
  rn_store<T, V>(q, o);
}
__device__ __forceinline__ u64 rn_all(float v) { return pk2(v, v); }
__device__ __forceinline__ u64 rn_neg1_plus(u64 v) { return fma2(v, rn_all(-1.f), rn_all(1.f)); }  // 1 - v
__device__ __forceinline__ u64 rn_sigmoid(u64 v) {
  const float2 t = upk2(mul2(v, rn_all(-LOG2E)));
  const float2 e = upk2(add2(pk2(ex2(t.x), ex2(t.y)), rn_all(1.f)));
  return pk2(rcp(e.x), rcp(e.y));
}
__device__ __forceinline__ float rn_hsum(u64 v) {
  const float2 t = upk2(v);
  return t.x + t.y;
}
// Bit i: channel c + i is kept (c and V multiples of 4).
template <int V>
__device__ __forceinline__ unsigned rn_bits(const RnParams& P, unsigned k0, unsigned k1, long long row, int c) {
  unsigned bits = 0;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const uint4 r = philox(make_uint4((unsigned)c / 4 + q, (unsigned)row, (unsigned)(row >> 32), P.offset), k0, k1);
    bits |= (r.x >= P.drop ? 1u : 0u) << (4 * q) | (r.y >= P.drop ? 2u : 0u) << (4 * q) |
            (r.z >= P.drop ? 4u : 0u) << (4 * q) | (r.w >= P.drop ? 8u : 0u) << (4 * q);
  }
  return P.drop_all ? 0u : bits;
}
__device__ __forceinline__ u64 rn_mask(u64 v, unsigned bits, int pair) {
  const float2 t = upk2(v);
  return pk2(bits >> (2 * pair) & 1 ? t.x : 0.f, bits >> (2 * pair + 1) & 1 ? t.y : 0.f);
}

template <typename TX, typename TO, int K>
__global__ void __launch_bounds__(512, 1) rn_fwd_ring_kernel(const __grid_constant__ RnParams P) {
  constexpr int V = 16 / sizeof(TO), H = V / 2;
  extern __shared__ __align__(128) char ring[];
  __shared__ float part[2][RN_MAX_WARPS];
  __shared__ uint64_t full[RN_MAX_GROUPS][RN_MAX_STAGES];
  const RnPlace a = rn_place<V>(P);
  const int rows = a.per * P.batch;
  const uint32_t xb = P.D * sizeof(TX), ob = P.D * sizeof(TO), row_bytes = xb + (P.g.p ? 2 : 1) * ob;
  char* stages = ring + (size_t)a.group * P.stages * rows * row_bytes;
  const unsigned long long seed = P.seed_ptr ? (unsigned long long)*P.seed_ptr : P.seed;
  const unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  const float inv = 1.f / P.D;
  if (a.mine == 0) {
    for (int q = 0; q < P.stages; ++q) rn_bar_init(&full[a.group][q]);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  bool alive = true;
  auto fetch = [&](long long row0, int s) {
    if (row0 >= P.rows || a.mine >= 32 || !alive) return;
    const int n = (int)min((long long)rows, P.rows - row0);
    uint64_t* bar = &full[a.group][s];
    char* d = stages + (size_t)s * rows * row_bytes;
    if (a.mine == 0) rn_expect(bar, n * row_bytes);
    rn_fetch<TX>(d, P.x, P.dense & 1, row0, n, P, bar);
    rn_fetch<TO>(d + (size_t)rows * xb, P.o, P.dense >> 1 & 1, row0, n, P, bar);
    if (P.g.p) rn_fetch<TO>(d + (size_t)rows * (xb + ob), P.g, P.dense >> 2 & 1, row0, n, P, bar);
  };
  for (int q = 0; q < P.stages; ++q) fetch(a.first + q * a.step, q);

  u64 w[K][H], wb[K][H], sc[K][H];  // the scale with 1 / (1 - p) in it
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = a.me * V + k * a.stride;
    const u64 keep = rn_all(P.dropout ? P.keep_scale : 1.f);
#pragma unroll
    for (int i = 0; i < H; ++i) w[k][i] = wb[k][i] = sc[k][i] = 0ull;
    if (c < P.D) {
      if (P.w) rn_get<float, V>(P.w + c, w[k]);
      if (P.wb) rn_get<float, V>(P.wb + c, wb[k]);
      if (P.scale) rn_get<float, V>(P.scale + c, sc[k]);
    }
#pragma unroll
    for (int i = 0; i < H; ++i) sc[k][i] = P.scale ? mul2(sc[k][i], keep) : keep;
  }
  const bool scaled = P.scale || P.dropout;
  int s = 0, turn = 0;
  for (long long row0 = a.first; row0 < P.rows; row0 += a.step) {
    if (alive) alive = rn_wait(&full[a.group][s], turn);
    const char* d = stages + (size_t)s * rows * row_bytes;
    for (int j = 0; j < P.batch; ++j) {
      const int at = j * a.per + a.sub;
      const long long row = row0 + at;
      if (row0 + j * a.per >= P.rows) break;  // (the whole group at once)
      const bool here = row < P.rows;
      const TX* px = reinterpret_cast<const TX*>(d) + (size_t)at * P.D;
      const TO* po = reinterpret_cast<const TO*>(d + (size_t)rows * xb) + (size_t)at * P.D;
      const TO* pg = reinterpret_cast<const TO*>(d + (size_t)rows * (xb + ob)) + (size_t)at * P.D;
      u64 v[K][H], ss = 0ull;
      float rb = 1.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = a.me * V + k * a.stride;
#pragma unroll
        for (int i = 0; i < H; ++i) v[k][i] = 0ull;
        if (c < P.D && here) {
          rn_get<TO, V>(po + c, v[k]);
#pragma unroll
          for (int i = 0; i < H; ++i) ss = fma2(v[k][i], v[k][i], ss);
        }
      }
      if (P.wb) {
        rb = rsqrtf(fmaf(rn_total(rn_hsum(ss), part, 0, a.group, P), inv, P.eps));
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], mul2(wb[k][i], rn_all(rb)));
      }
      ss = 0ull;
      TX* pv = static_cast<TX*>(P.v) + row * P.D;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = a.me * V + k * a.stride;
        if (c < P.D && here) {
          u64 f[H];
          if (P.g.p) {
            rn_get<TO, V>(pg + c, f);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], rn_sigmoid(f[i]));
          }
          if (scaled)
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], sc[k][i]);
          if (P.dropout) {
            const unsigned bits = rn_bits<V>(P, k0, k1, row, c);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = rn_mask(v[k][i], bits, i);
          }
          rn_get<TX, V>(px + c, f);
#pragma unroll
          for (int i = 0; i < H; ++i) {
            v[k][i] = add2(v[k][i], f[i]);
            ss = fma2(v[k][i], v[k][i], ss);
          }
          rn_put<TX, V>(pv + c, v[k]);
        }
      }
      float r = 0.f;
      if (P.w) {
        r = rsqrtf(fmaf(rn_total(rn_hsum(ss), part, 1, a.group, P), inv, P.eps));
        TO* pn = static_cast<TO*>(P.n) + row * P.D;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = a.me * V + k * a.stride;
          if (c < P.D && here) {
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], mul2(w[k][i], rn_all(r)));
            rn_put<TO, V>(pn + c, v[k]);
          }
        }
      }
      if (P.rstd && a.me == 0 && here) *reinterpret_cast<float2*>(P.rstd + 2 * row) = make_float2(rb, r);
      // everyone has read the row (two sums: the second one's barrier says so, and keeps their slots apart)
      if (P.warps == 1) __syncwarp();
      else if (!P.w || !P.wb) asm volatile("bar.sync %0, %1;" ::"r"(a.group + 1), "r"(P.warps * 32) : "memory");
    }
    fetch(row0 + P.stages * a.step, s);
    if (++s == P.stages) s = 0, turn ^= 1;
  }
  if (!alive) {  // a copy did not arrive: report it, and let what is in flight land (waiting again, as long)
    atomicExch(P.err, 12);
    if (a.mine == 0)
      for (int q = 0; q < P.stages; ++q) rn_wait(&full[a.group][q], q < s ? turn ^ 1 : turn);
  }
}

template <typename TX, typename TO, int K>
__global__ void __launch_bounds__(512, 1) rn_bwd_ring_kernel(const __grid_constant__ RnParams P) {
  constexpr int V = 16 / sizeof(TO), H = V / 2;
  extern __shared__ __align__(128) char ring[];  // the parameters [3][D], then the groups' stages
  __shared__ float part[2][RN_MAX_WARPS];
  __shared__ uint64_t full[RN_MAX_GROUPS][RN_MAX_STAGES];
  const RnPlace a = rn_place<V>(P);
  const int rows = a.per * P.batch;
  const bool has_g = P.g.p != nullptr, has_dv = P.dv.p != nullptr, has_dn = P.dn.p != nullptr;
  const uint32_t xb = P.D * sizeof(TX), ob = P.D * sizeof(TO);
  const uint32_t off_o = xb, off_g = off_o + ob, off_dv = off_g + (has_g ? ob : 0), off_dn = off_dv + (has_dv ? xb : 0);
  const uint32_t row_bytes = off_dn + (has_dn ? ob : 0);
  float* params = reinterpret_cast<float*>(ring);
  char* stages = ring + (size_t)3 * P.D * 4 + (size_t)a.group * P.stages * rows * row_bytes;
  const unsigned long long seed = P.seed_ptr ? (unsigned long long)*P.seed_ptr : P.seed;
  const unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  const float inv = 1.f / P.D;
  if (a.mine == 0) {
    for (int q = 0; q < P.stages; ++q) rn_bar_init(&full[a.group][q]);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = threadIdx.x; i < P.D; i += blockDim.x) {
    params[i] = P.w ? P.w[i] : 0.f;
    params[P.D + i] = P.wb ? P.wb[i] : 1.f;
    params[2 * P.D + i] = (P.scale ? P.scale[i] : 1.f) * (P.dropout ? P.keep_scale : 1.f);
  }
  __syncthreads();

  bool alive = true;
  auto fetch = [&](long long row0, int s) {
    if (row0 >= P.rows || a.mine >= 32 || !alive) return;
    const int n = (int)min((long long)rows, P.rows - row0);
    uint64_t* bar = &full[a.group][s];
    char* d = stages + (size_t)s * rows * row_bytes;
    if (a.mine == 0) rn_expect(bar, n * row_bytes);
    rn_fetch<TX>(d, P.x, P.dense & 1, row0, n, P, bar);
    rn_fetch<TO>(d + (size_t)rows * off_o, P.o, P.dense >> 1 & 1, row0, n, P, bar);
    if (has_g) rn_fetch<TO>(d + (size_t)rows * off_g, P.g, P.dense >> 2 & 1, row0, n, P, bar);
    if (has_dv) rn_fetch<TX>(d + (size_t)rows * off_dv, P.dv, P.dense >> 3 & 1, row0, n, P, bar);
    if (has_dn) rn_fetch<TO>(d + (size_t)rows * off_dn, P.dn, P.dense >> 4 & 1, row0, n, P, bar);
  };
  for (int q = 0; q < P.stages; ++q) fetch(a.first + q * a.step, q);

  u64 sw[K][H], sb[K][H], ssc[K][H];  // sums over this thread's rows
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < H; ++i) sw[k][i] = sb[k][i] = ssc[k][i] = 0ull;
  const float keep = P.dropout ? P.keep_scale : 1.f;
  int s = 0, turn = 0;
  for (long long row0 = a.first; row0 < P.rows; row0 += a.step) {
    if (alive) alive = rn_wait(&full[a.group][s], turn);
    const char* d = stages + (size_t)s * rows * row_bytes;
    for (int j = 0; j < P.batch; ++j) {
      const int at = j * a.per + a.sub;
      const long long row = row0 + at;
      if (row0 + j * a.per >= P.rows) break;
      const bool here = row < P.rows;
      const TX* px = reinterpret_cast<const TX*>(d) + (size_t)at * P.D;
      const TO* po = reinterpret_cast<const TO*>(d + (size_t)rows * off_o) + (size_t)at * P.D;
      const TO* pg = reinterpret_cast<const TO*>(d + (size_t)rows * off_g) + (size_t)at * P.D;
      const TX* pdv = reinterpret_cast<const TX*>(d + (size_t)rows * off_dv) + (size_t)at * P.D;
      const TO* pdn = reinterpret_cast<const TO*>(d + (size_t)rows * off_dn) + (size_t)at * P.D;
      const float2 roots = here ? *reinterpret_cast<const float2*>(P.rstd + 2 * row) : make_float2(0.f, 0.f);
      const float rb = roots.x, r = roots.y;
      // the stream again, and the next norm's sum of t v
      u64 v[K][H], dot = 0ull;
      unsigned bits[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = a.me * V + k * a.stride;
        bits[k] = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < H; ++i) v[k][i] = 0ull;
        if (c < P.D && here) {
          u64 f[H];
          if (P.dropout) bits[k] = rn_bits<V>(P, k0, k1, row, c);
          if (has_dn) {
            rn_get<TO, V>(po + c, v[k]);
            rn_get<float, V>(params + P.D + c, f);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], mul2(f[i], rn_all(rb)));
            if (has_g) {
              rn_get<TO, V>(pg + c, f);
#pragma unroll
              for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], rn_sigmoid(f[i]));
            }
            rn_get<float, V>(params + 2 * P.D + c, f);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], f[i]);
            if (P.dropout)
#pragma unroll
              for (int i = 0; i < H; ++i) v[k][i] = rn_mask(v[k][i], bits[k], i);
            rn_get<TX, V>(px + c, f);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = add2(v[k][i], f[i]);
            u64 t[H];
            rn_get<TO, V>(pdn + c, t);
            rn_get<float, V>(params + c, f);
#pragma unroll
            for (int i = 0; i < H; ++i) dot = fma2(mul2(t[i], f[i]), v[k][i], dot);
          }
        }
      }
      float mean = 0.f;
      if (has_dn) mean = rn_total(rn_hsum(dot), part, 0, a.group, P) * inv * r * r;
      dot = 0ull;
      TX* pdx = static_cast<TX*>(P.dx) + row * P.D;
      TO* pdg = static_cast<TO*>(P.dg) + row * P.D;
      TO* pdo = static_cast<TO*>(P.d_o) + row * P.D;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = a.me * V + k * a.stride;
        if (c < P.D && here) {
          u64 g[H], f[H], t[H];  // g: gradient of the stream
          if (has_dn) {
            rn_get<TO, V>(pdn + c, t);
            rn_get<float, V>(params + c, f);
#pragma unroll
            for (int i = 0; i < H; ++i) {
              g[i] = mul2(rn_all(r), fma2(v[k][i], rn_all(-mean), mul2(f[i], t[i])));
              sw[k][i] = fma2(mul2(t[i], v[k][i]), rn_all(r), sw[k][i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < H; ++i) g[i] = 0ull;
          }
          if (has_dv) {
            rn_get<TX, V>(pdv + c, f);
#pragma unroll
            for (int i = 0; i < H; ++i) g[i] = add2(g[i], f[i]);
          }
          rn_put<TX, V>(pdx + c, g);
          if (P.dropout)
#pragma unroll
            for (int i = 0; i < H; ++i) g[i] = rn_mask(g[i], bits[k], i);
          u64 u[H], sg[H];
          rn_get<TO, V>(po + c, u);
          rn_get<float, V>(params + P.D + c, f);
          if (has_g) rn_get<TO, V>(pg + c, sg);
          rn_get<float, V>(params + 2 * P.D + c, t);
#pragma unroll
          for (int i = 0; i < H; ++i) {
            const u64 n = mul2(u[i], rn_all(rb));        // the branch, normed
            const u64 ui = mul2(n, f[i]);
            const u64 si = has_g ? rn_sigmoid(sg[i]) : rn_all(1.f);
            u64 us = mul2(ui, si);
            if (P.dropout) us = rn_mask(us, bits[k], i);  // a dropped element may hold anything
            if (P.scale) ssc[k][i] = fma2(mul2(g[i], us), rn_all(keep), ssc[k][i]);
            const u64 ds = mul2(g[i], t[i]);              // of u s
            if (has_g) sg[i] = mul2(mul2(ds, us), rn_neg1_plus(si));
            u64 du = mul2(ds, si);
            if (P.dropout) {
              du = rn_mask(du, bits[k], i);
              if (has_g) sg[i] = rn_mask(sg[i], bits[k], i);
            }
            if (P.wb) {
              sb[k][i] = fma2(du, n, sb[k][i]);
              du = mul2(du, f[i]);
              dot = fma2(du, u[i], dot);
            }
            v[k][i] = du;
          }
          if (has_g) rn_put<TO, V>(pdg + c, sg);
          if (!P.wb) rn_put<TO, V>(pdo + c, v[k]);
        }
      }
      if (P.wb) {
        mean = rn_total(rn_hsum(dot), part, 1, a.group, P) * inv * rb * rb;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = a.me * V + k * a.stride;
          if (c < P.D && here) {
            u64 u[H];
            rn_get<TO, V>(po + c, u);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = mul2(rn_all(rb), fma2(u[i], rn_all(-mean), v[k][i]));
            rn_put<TO, V>(pdo + c, v[k]);
          }
        }
      }
      // everyone has read the row, and the sums' slots may be written again
      if (P.warps == 1) __syncwarp();
      else asm volatile("bar.sync %0, %1;" ::"r"(a.group + 1), "r"(P.warps * 32) : "memory");
    }
    fetch(row0 + P.stages * a.step, s);
    if (++s == P.stages) s = 0, turn ^= 1;
  }
  if (!alive) {
    atomicExch(P.err, 12);
    if (a.mine == 0)
      for (int q = 0; q < P.stages; ++q) rn_wait(&full[a.group][q], q < s ? turn ^ 1 : turn);
  }
  // the CTA's sums: its threads of a channel in order (groups, then rows at once), through the parameters' place
  __syncthreads();
  float* out = P.partial + (long long)blockIdx.x * 3 * P.D;
  const int groups = (int)(blockDim.x >> 5) / P.warps;
  for (int q = 0; q < groups * a.per; ++q) {
    if (a.group == q / a.per && a.sub == q % a.per)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = a.me * V + k * a.stride;
        if (c < P.D)
#pragma unroll
          for (int i = 0; i < H; ++i) {
            u64* f0 = reinterpret_cast<u64*>(params + c) + i;
            u64* f1 = reinterpret_cast<u64*>(params + P.D + c) + i;
            u64* f2 = reinterpret_cast<u64*>(params + 2 * P.D + c) + i;
            *f0 = q ? add2(*f0, sw[k][i]) : sw[k][i];
            *f1 = q ? add2(*f1, sb[k][i]) : sb[k][i];
            *f2 = q ? add2(*f2, ssc[k][i]) : ssc[k][i];
          }
      }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 3 * P.D; i += blockDim.x) out[i] = params[i];
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
