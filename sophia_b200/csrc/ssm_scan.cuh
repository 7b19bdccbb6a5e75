// Selective state space scan.  Per sequence, channel e and state n:
//   d[t] = softplus(dt[t] + dt_bias)  (or dt + dt_bias),  a[t] = e^(d[t] A[n]),
//   h[t] = a[t] h[t-1] + d[t] x[t] B[t][n],
//   s[t] = sum_n C[t][n] h[t][n] + D x[t],   y[t] = s[t] silu(z[t])  (or s[t]),
// h before the first token being the initial state (zeros without one).  B and
// C are shared by the channels of a group.  Backward, with ds = dy silu(z):
//   g[t] = C[t] ds[t] + a[t+1] g[t+1]   (plus the final state's gradient at the end),
//   dC[t][n] = sum_e ds h,   dB[t][n] = sum_e g d x,   q = a g h[t-1],
//   dd = sum_n q A + x sum_n g B,   dx = d sum_n g B + D ds,   dA = sum_t q d,
//   dz = dy s silu'(z),   d dt = dd softplus',   dD = sum_t ds x.
//
// Layout.  Time runs over lanes: a lane owns K = 8 consecutive tokens of two
// neighbouring channels (one fp32 pair in packed arithmetic), LT lanes make
// a tile of 8 LT tokens, 32 / LT channel pairs share a warp.  Per state, a lane
// composes its tokens' steps to (decay, value), the LT lanes combine theirs by a
// shuffle scan that starts from the state carried over the tiles, and a second
// pass over the tokens gives h.  So each decay's exponential is evaluated once and
// a tile needs no step-by-step pass; B and C rows are shared by all lanes of a
// token; and in the backward the sums over channels in dB and dC are, in each
// lane, sums over the channels that its warp takes, for fixed tokens.
// Tiles of x, dt, z (and dy) are staged in shared memory, rows of one token
// skewed by 16 bytes per 8 tokens so that lanes 8 tokens apart use other banks.
#pragma once

#include <type_traits>

#include "ssm_common.cuh"

namespace kda {

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
__device__ __forceinline__ u64 ex2_2(u64 a) {
  const float2 v = upk2(a);
  return pk2(ex2(v.x), ex2(v.y));
}

constexpr int SCAN_K = 8;          // tokens per lane
constexpr int SCAN_THREADS = 256;  // 8 warps
constexpr int SCAN_WARPS = SCAN_THREADS / 32;

// Geometry of a variant with LT lanes along time and elements of T.
template <typename T, int LT>
struct ScanGeo {
  static constexpr int TL = LT * SCAN_K;                   // tokens per tile
  static constexpr int CL = 32 / LT;                       // channel pairs per warp
  static constexpr int CPB = SCAN_WARPS * CL * 2;          // channels per CTA
  static constexpr int ROWB = CPB * (int)sizeof(T);        // bytes of a staged row
  static constexpr int RAW = TL * ROWB + (TL / 8) * 16;    // bytes of a staged tensor
  static constexpr int BCP = TL + 4;                       // floats per state of staged B or C
  static __host__ __device__ int raw_off(int t, int c) { return t * ROWB + (t >> 3) * 16 + c * (int)sizeof(T); }
  // B and C: tokens 8l .. 8l+3 of every lane l first, then 8l+4 .. 8l+7, so that a
  // lane's two 16-byte reads are conflict-free
  static __host__ __device__ int bc_off(int t) { return ((t >> 2) & 1) * (TL / 2) + (t >> 3) * 4 + (t & 3); }
};

struct ScanParams {
  RowView x, dt, z, dy;            // [B, T, E]; z.p null = no gate
  const void *Bm, *Cm;             // [B, T, G, N], rows of N contiguous
  long long b_sb, b_st, b_sg, c_sb, c_st, c_sg;
  const float *A, *D, *dt_bias;    // [E][N], [E] or null, [E] or null
  const float* h0;                 // [nseq][E][N] or null
  SeqMap seq;
  int B, T, E, N, G;
  int tiles, blocks;               // tiles per row, channel blocks per group
  bool softplus, vec;              // vec: 16-byte staging is aligned for x, dt, z, dy and the outputs
  void* y;                         // [B, T, E] contiguous
  float* ht;                       // [nseq][E][N] or null
  float* ckpt;                     // [B][tiles][G * blocks][N][CPB] states at the tiles' starts, or null
  // backward
  const float* dht;
  void *dx, *ddt, *dz;
  float* dh0;
  float* bc_part;                  // [B][tiles][G][blocks][2][N][TL]
  float* e_part;                   // [B][E][N + 2]: dA, dD, d dt_bias
};

struct ScanBlock {
  int g, blk, c0, nc, b;  // group, block in it, first channel, channels, row
};
template <int CPB>
__device__ __forceinline__ ScanBlock scan_block(const ScanParams& P) {
  ScanBlock s;
  const int eg = P.E / P.G;
  s.g = blockIdx.x / P.blocks;
  s.blk = blockIdx.x - s.g * P.blocks;
  s.c0 = s.g * eg + s.blk * CPB;
  s.nc = min(CPB, eg - s.blk * CPB);
  s.b = blockIdx.y;
  return s;
}

// Stages rows t0 .. t0+TL-1 (zeros past T and past the block's channels).
template <typename T, int LT>
__device__ __forceinline__ void scan_stage(char* dst, const RowView& r, const ScanParams& P, const ScanBlock& s, int t0) {
  using G = ScanGeo<T, LT>;
  constexpr int V = 16 / (int)sizeof(T), NV = G::CPB / V;
  if (P.vec) {
#pragma unroll 4
    for (int i = threadIdx.x; i < G::TL * NV; i += SCAN_THREADS) {
      const int t = i / NV, c = (i - t * NV) * V;
      IoVec<T, V> v;
#pragma unroll
      for (int k = 0; k < V; ++k) v.v[k] = io_from_f<T>(0.f);
      if (t0 + t < P.T) {
        const T* p = row_ptr<T>(r, s.b, t0 + t) + s.c0 + c;
        if (c + V <= s.nc) {
          v = *reinterpret_cast<const IoVec<T, V>*>(p);
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (c + k < s.nc) v.v[k] = p[k];
        }
      }
      *reinterpret_cast<IoVec<T, V>*>(dst + G::raw_off(t, c)) = v;
    }
  } else {
    for (int i = threadIdx.x; i < G::TL * G::CPB; i += SCAN_THREADS) {
      const int t = i / G::CPB, c = i - t * G::CPB;
      T v = io_from_f<T>(0.f);
      if (t0 + t < P.T && c < s.nc) v = row_ptr<T>(r, s.b, t0 + t)[s.c0 + c];
      *reinterpret_cast<T*>(dst + G::raw_off(t, c)) = v;
    }
  }
}

// Writes a staged tile to a contiguous [B, T, E] output.
template <typename T, int LT>
__device__ __forceinline__ void scan_unstage(const char* src, void* out, const ScanParams& P, const ScanBlock& s, int t0) {
  using G = ScanGeo<T, LT>;
  constexpr int V = 16 / (int)sizeof(T), NV = G::CPB / V;
  T* base = static_cast<T*>(out) + ((long long)s.b * P.T + t0) * P.E + s.c0;
  if (P.vec) {
    for (int i = threadIdx.x; i < G::TL * NV; i += SCAN_THREADS) {
      const int t = i / NV, c = (i - t * NV) * V;
      if (t0 + t >= P.T || c >= s.nc) continue;
      const IoVec<T, V> v = *reinterpret_cast<const IoVec<T, V>*>(src + G::raw_off(t, c));
      T* p = base + (long long)t * P.E + c;
      if (c + V <= s.nc) {
        *reinterpret_cast<IoVec<T, V>*>(p) = v;
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (c + k < s.nc) p[k] = v.v[k];
      }
    }
  } else {
    for (int i = threadIdx.x; i < G::TL * G::CPB; i += SCAN_THREADS) {
      const int t = i / G::CPB, c = i - t * G::CPB;
      if (t0 + t < P.T && c < s.nc) base[(long long)t * P.E + c] = *reinterpret_cast<const T*>(src + G::raw_off(t, c));
    }
  }
}

// Stages B or C of a tile as fp32 [N][BCP] (zeros past T).
template <typename T, int LT>
__device__ __forceinline__ void scan_stage_bc(float* dst, const void* src, long long sb, long long st, long long sg,
                                              const ScanParams& P, const ScanBlock& s, int t0, int np2) {
  using G = ScanGeo<T, LT>;
  const T* p = static_cast<const T*>(src) + s.b * sb + s.g * sg;
  const int n = threadIdx.x & (np2 - 1);  // np2: the power of two at or above N
  if (n >= P.N) return;
  const int step = SCAN_THREADS / np2;
#pragma unroll 4
  for (int t = threadIdx.x / np2; t < G::TL; t += step)
    dst[n * G::BCP + G::bc_off(t)] = t0 + t < P.T ? io_to_f(p[(long long)(t0 + t) * st + n]) : 0.f;
}

template <typename T>
__device__ __forceinline__ u64 scan_pair(const char* p) {
  const IoVec<T, 2> v = *reinterpret_cast<const IoVec<T, 2>*>(p);
  return pk2(io_to_f(v.v[0]), io_to_f(v.v[1]));
}
template <typename T>
__device__ __forceinline__ void scan_put(char* p, float2 v) {
  IoVec<T, 2> r;
  r.v[0] = io_from_f<T>(v.x);
  r.v[1] = io_from_f<T>(v.y);
  *reinterpret_cast<IoVec<T, 2>*>(p) = r;
}

__device__ __forceinline__ void scan_row8(const float* base, int half, int tl, float (&v)[SCAN_K]) {
  const float4 a = *reinterpret_cast<const float4*>(base + tl * 4);
  const float4 b = *reinterpret_cast<const float4*>(base + half + tl * 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

template <int LT>
__device__ __forceinline__ u64 scan_up(u64 v, int off) { return __shfl_up_sync(0xffffffffu, v, off, LT); }
template <int LT>
__device__ __forceinline__ u64 scan_down(u64 v, int off) { return __shfl_down_sync(0xffffffffu, v, off, LT); }

// Inclusive scan over the LT lanes of h <- p h_before + h, p being the lane's own
// decay.  RESET: bit k of `block` stops what comes in step k, because a sequence starts in
// the span on this side of it (selected away, not multiplied by zero: another
// sequence's infinities and NaN stay its own).
template <int LT, bool RESET>
__device__ __forceinline__ void scan_lanes(u64& h, u64 p, int tl, unsigned block) {
#pragma unroll
  for (int off = 1, k = 0; off < LT; off <<= 1, ++k) {
    const u64 hn = scan_up<LT>(h, off);
    const bool take = tl >= off && !(RESET && (block >> k & 1));
    if (off * 2 < LT) {
      const u64 pn = scan_up<LT>(p, off);
      if (take) {
        h = fma2(p, hn, h);
        p = mul2(p, pn);
      }
    } else if (take) {
      h = fma2(p, hn, h);
    }
  }
}
// The same towards lower lanes.
template <int LT, bool RESET>
__device__ __forceinline__ void scan_lanes_rev(u64& h, u64 p, int tl, unsigned block) {
#pragma unroll
  for (int off = 1, k = 0; off < LT; off <<= 1, ++k) {
    const u64 hn = scan_down<LT>(h, off);
    const bool take = tl + off < LT && !(RESET && (block >> k & 1));
    if (off * 2 < LT) {
      const u64 pn = scan_down<LT>(p, off);
      if (take) {
        h = fma2(p, hn, h);
        p = mul2(p, pn);
      }
    } else if (take) {
      h = fma2(p, hn, h);
    }
  }
}

// Where sequences start and end among a lane's tokens (bit j: token j), and which
// steps of the two lane scans that stops.
struct ScanFlags {
  unsigned first, last, up, down;
  bool any_first, any_last;  // anywhere in the tile
};
template <int LT>
__device__ __forceinline__ ScanFlags scan_flags(const int* first, const int* last, int tl) {
  ScanFlags f{};
#pragma unroll
  for (int j = 0; j < SCAN_K; ++j) {
    f.first |= (unsigned)(first[tl * SCAN_K + j] >= 0) << j;
    f.last |= (unsigned)(last[tl * SCAN_K + j] >= 0) << j;
  }
  const unsigned starts = __ballot_sync(0xffffffffu, f.first != 0);
  f.any_first = starts != 0;
  f.any_last = __ballot_sync(0xffffffffu, f.last != 0) != 0;
  const unsigned mine = LT == 32 ? starts : (starts >> ((threadIdx.x & 31) / LT * LT)) & ((1u << (LT & 31)) - 1u);
#pragma unroll
  for (int off = 1, k = 0; off < LT; off <<= 1, ++k) {
    const unsigned span = (1u << off) - 1u;  // off <= 16
    if (tl >= off && ((mine >> (tl - off + 1)) & span)) f.up |= 1u << k;
    if ((mine >> tl) & span) f.down |= 1u << k;
  }
  return f;
}

// Sum over the LT lanes of a channel pair.
template <int LT>
__device__ __forceinline__ u64 scan_sum(u64 v) {
#pragma unroll
  for (int m = LT / 2; m >= 1; m >>= 1) v = add2(v, __shfl_xor_sync(0xffffffffu, v, m, LT));
  return v;
}

// A lane's steps d (0 past T), inputs d x, the sum of d, and the flags of its
// tokens that are a sequence's first or last.
template <typename T, int LT>
__device__ __forceinline__ void scan_inputs(const ScanParams& P, const char* rx, const char* rdt, int t0, int tl, int c,
                                            u64 bias, u64 (&d)[SCAN_K], u64 (&u)[SCAN_K], u64& sum) {
  using G = ScanGeo<T, LT>;
  sum = pk2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < SCAN_K; ++j) {
    const int t = tl * SCAN_K + j;
    const float2 r = upk2(add2(scan_pair<T>(rdt + G::raw_off(t, c)), bias));
    u64 v = P.softplus ? pk2(softplusf_(r.x), softplusf_(r.y)) : pk2(r.x, r.y);
    if (t0 + t >= P.T) v = pk2(0.f, 0.f);
    d[j] = v;
    u[j] = mul2(v, scan_pair<T>(rx + G::raw_off(t, c)));
    sum = add2(sum, v);
  }
}

// Shared memory: staged tensors, B, C, log2-scaled A, the carried states and the
// sequence flags of the tile (packed).  The backward adds the carried gradients, the
// dB and dC of the tile and the lanes' dA sums.
template <typename T, int LT>
__host__ __device__ inline int scan_smem_bytes(int N, int tensors, bool bwd) {
  using G = ScanGeo<T, LT>;
  int b = tensors * G::RAW + 2 * N * G::BCP * 4 + 2 * N * G::CPB * 4 + 2 * G::TL * 4;
  if (bwd) b += N * G::CPB * 4 + 2 * N * G::TL * 4 + N * (LT == 32 ? SCAN_THREADS * 8 : G::CPB * 4);
  return b;
}

__device__ __forceinline__ float2 scan_state2(const float* p, long long row, int E, int N, int c, int nc, int c0, int n) {
  float2 v = make_float2(0.f, 0.f);
  const float* q = p + (row * E + c0 + c) * (long long)N + n;
  if (c < nc) v.x = __ldg(q);
  if (c + 1 < nc) v.y = __ldg(q + N);
  return v;
}
__device__ __forceinline__ void scan_put_state2(float* p, long long row, int E, int N, int c, int nc, int c0, int n,
                                                float2 v) {
  float* q = p + (row * E + c0 + c) * (long long)N + n;
  if (c < nc) q[0] = v.x;
  if (c + 1 < nc) q[N] = v.y;
}

template <typename T, int LT, bool PACKED>
__global__ void __launch_bounds__(SCAN_THREADS) ssm_scan_fwd_kernel(ScanParams P, int np2) {
  using G = ScanGeo<T, LT>;
  extern __shared__ __align__(16) char scan_sm[];
  char* rx = scan_sm;
  char* rdt = rx + G::RAW;
  char* rz = rdt + G::RAW;
  float* Bs = reinterpret_cast<float*>(rz + (P.z.p ? G::RAW : 0));
  float* Cs = Bs + P.N * G::BCP;
  float* A2 = Cs + P.N * G::BCP;       // [N][CPB]
  float* carry = A2 + P.N * G::CPB;    // [N][CPB]
  int* first = reinterpret_cast<int*>(carry + P.N * G::CPB);  // [TL]
  int* last = first + G::TL;

  const ScanBlock s = scan_block<G::CPB>(P);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tl = lane % LT, c = warp * (2 * G::CL) + (lane / LT) * 2;
  const int N = P.N;
  for (int i = threadIdx.x; i < N * G::CPB; i += SCAN_THREADS) {
    const int n = i / G::CPB, cc = i - n * G::CPB;
    const bool ok = cc < s.nc;
    A2[i] = ok ? P.A[(long long)(s.c0 + cc) * N + n] * LOG2E : 0.f;
    carry[i] = !PACKED && P.h0 && ok ? P.h0[((long long)s.b * P.E + s.c0 + cc) * N + n] : 0.f;
  }
  const float2 zero2 = make_float2(0.f, 0.f);
  float2 bias = zero2, dskip = zero2;
  if (c < s.nc) {
    if (P.dt_bias) bias.x = P.dt_bias[s.c0 + c];
    if (P.D) dskip.x = P.D[s.c0 + c];
  }
  if (c + 1 < s.nc) {
    if (P.dt_bias) bias.y = P.dt_bias[s.c0 + c + 1];
    if (P.D) dskip.y = P.D[s.c0 + c + 1];
  }
  const u64 bias2 = pk2(bias.x, bias.y);

  for (int tile = 0; tile < P.tiles; ++tile) {
    const int t0 = tile * G::TL;
    __syncthreads();  // the tile in front has left
    scan_stage<T, LT>(rx, P.x, P, s, t0);
    scan_stage<T, LT>(rdt, P.dt, P, s, t0);
    if (P.z.p) scan_stage<T, LT>(rz, P.z, P, s, t0);
    scan_stage_bc<T, LT>(Bs, P.Bm, P.b_sb, P.b_st, P.b_sg, P, s, t0, np2);
    scan_stage_bc<T, LT>(Cs, P.Cm, P.c_sb, P.c_st, P.c_sg, P, s, t0, np2);
    if (PACKED) {
      for (int i = threadIdx.x; i < G::TL; i += SCAN_THREADS) {
        first[i] = t0 + i < P.T ? __ldg(P.seq.start + t0 + i) : -1;
        last[i] = t0 + i < P.T ? __ldg(P.seq.end + t0 + i) : -1;
      }
    }
    if (P.ckpt) {
      float* ck = P.ckpt + (((long long)s.b * P.tiles + tile) * gridDim.x + blockIdx.x) * (N * G::CPB);
      for (int i = threadIdx.x; i < N * G::CPB; i += SCAN_THREADS) ck[i] = carry[i];
    }
    __syncthreads();

    u64 d[SCAN_K], u[SCAN_K], y[SCAN_K], sum;
    scan_inputs<T, LT>(P, rx, rdt, t0, tl, c, bias2, d, u, sum);
    ScanFlags f{};
    if (PACKED) f = scan_flags<LT>(first, last, tl);
#pragma unroll
    for (int j = 0; j < SCAN_K; ++j) y[j] = pk2(0.f, 0.f);

    auto states = [&](auto reset) {
      constexpr bool RESET = decltype(reset)::value;
#pragma unroll 1
      for (int n = 0; n < N; ++n) {
        const u64 a2 = *reinterpret_cast<const u64*>(A2 + n * G::CPB + c);
        const u64 h_in = *reinterpret_cast<const u64*>(carry + n * G::CPB + c);
        float bv[SCAN_K], cv[SCAN_K];
        scan_row8(Bs + n * G::BCP, G::TL / 2, tl, bv);
        scan_row8(Cs + n * G::BCP, G::TL / 2, tl, cv);
        u64 a[SCAN_K], b[SCAN_K];
#pragma unroll
        for (int j = 0; j < SCAN_K; ++j) {
          a[j] = ex2_2(mul2(d[j], a2));
          b[j] = mul2(u[j], pk2(bv[j], bv[j]));
        }
        if (RESET && P.h0) {  // a sequence's first token takes up its initial state
#pragma unroll
          for (int j = 0; j < SCAN_K; ++j)
            if (f.first >> j & 1) {
              const float2 h = scan_state2(P.h0, first[tl * SCAN_K + j], P.E, N, c, s.nc, s.c0, n);
              b[j] = fma2(a[j], pk2(h.x, h.y), b[j]);
            }
        }
        u64 h = b[0];
#pragma unroll
        for (int j = 1; j < SCAN_K; ++j) h = RESET && (f.first >> j & 1) ? b[j] : fma2(a[j], h, b[j]);
        const u64 p = ex2_2(mul2(sum, a2));
        if (tl == 0 && !(RESET && f.first)) h = fma2(p, h_in, h);
        scan_lanes<LT, RESET>(h, p, tl, f.up);
        __syncwarp();  // every lane has read the carried state
        if (tl == LT - 1) *reinterpret_cast<u64*>(carry + n * G::CPB + c) = h;
        h = scan_up<LT>(h, 1);
        if (tl == 0) h = h_in;
#pragma unroll
        for (int j = 0; j < SCAN_K; ++j) {
          h = RESET && (f.first >> j & 1) ? b[j] : fma2(a[j], h, b[j]);
          if (PACKED) b[j] = h;
          y[j] = fma2(h, pk2(cv[j], cv[j]), y[j]);
        }
        if (PACKED && f.any_last && P.ht) {
#pragma unroll
          for (int j = 0; j < SCAN_K; ++j)
            if (f.last >> j & 1)
              scan_put_state2(P.ht, last[tl * SCAN_K + j], P.E, N, c, s.nc, s.c0, n, upk2(b[j]));
        }
      }
    };
    if (PACKED && f.any_first) states(std::true_type{});
    else states(std::false_type{});

    const u64 skip2 = pk2(dskip.x, dskip.y);
#pragma unroll
    for (int j = 0; j < SCAN_K; ++j) {
      const int off = G::raw_off(tl * SCAN_K + j, c);
      float2 v = upk2(fma2(skip2, scan_pair<T>(rx + off), y[j]));
      if (P.z.p) {
        const float2 z = upk2(scan_pair<T>(rz + off));
        v.x *= siluf_(z.x);
        v.y *= siluf_(z.y);
      }
      scan_put<T>(rx + off, v);
    }
    __syncthreads();
    scan_unstage<T, LT>(rx, P.y, P, s, t0);
  }
  if (!PACKED && P.ht)
    for (int i = threadIdx.x; i < N * G::CPB; i += SCAN_THREADS) {
      const int n = i / G::CPB, cc = i - n * G::CPB;
      if (cc < s.nc) P.ht[((long long)s.b * P.E + s.c0 + cc) * N + n] = carry[i];
    }
}

// Backward: tiles from last to first; each rebuilds its states from the forward's
// state at the tile's start.  The eight warps take the states n in an order of their
// own (warp w starts at n = w), one barrier per step, so that no two add to the same dB
// and dC rows at once and every sum has a fixed order.
template <typename T, int LT, bool PACKED>
__global__ void __launch_bounds__(SCAN_THREADS) ssm_scan_bwd_kernel(ScanParams P, int np2) {
  using G = ScanGeo<T, LT>;
  extern __shared__ __align__(16) char scan_sm[];
  char* rx = scan_sm;
  char* rdt = rx + G::RAW;
  char* rdy = rdt + G::RAW;
  char* rz = rdy + G::RAW;
  float* Bs = reinterpret_cast<float*>(rz + (P.z.p ? G::RAW : 0));
  float* Cs = Bs + P.N * G::BCP;
  float* A2 = Cs + P.N * G::BCP;
  float* hst = A2 + P.N * G::CPB;     // states at the tile's start
  float* gcar = hst + P.N * G::CPB;   // gradient of the state in front of the tile behind
  float* dBs = gcar + P.N * G::CPB;   // [2][N][TL], tokens in bc_off order
  // dA: a sum per lane over the tiles with 32 lanes on time ([N][threads]), a sum per
  // channel pair with fewer (three shuffles a state; [N][CPB])
  constexpr int DAW = LT == 32 ? SCAN_THREADS : G::CPB / 2;
  u64* dAs = reinterpret_cast<u64*>(dBs + 2 * P.N * G::TL);
  int* first = reinterpret_cast<int*>(dAs + P.N * DAW);
  int* last = first + G::TL;

  const ScanBlock s = scan_block<G::CPB>(P);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tl = lane % LT, c = warp * (2 * G::CL) + (lane / LT) * 2;
  const int N = P.N, steps = max(N, SCAN_WARPS);
  float* dCs = dBs + N * G::TL;
  for (int i = threadIdx.x; i < N * G::CPB; i += SCAN_THREADS) {
    const int n = i / G::CPB, cc = i - n * G::CPB;
    const bool ok = cc < s.nc;
    A2[i] = ok ? P.A[(long long)(s.c0 + cc) * N + n] * LOG2E : 0.f;
    gcar[i] = !PACKED && P.dht && ok ? P.dht[((long long)s.b * P.E + s.c0 + cc) * N + n] : 0.f;
  }
  for (int i = threadIdx.x; i < N * DAW; i += SCAN_THREADS) dAs[i] = 0;
  const float2 zero2 = make_float2(0.f, 0.f);
  float2 bias = zero2, dskip = zero2;
  if (c < s.nc) {
    if (P.dt_bias) bias.x = P.dt_bias[s.c0 + c];
    if (P.D) dskip.x = P.D[s.c0 + c];
  }
  if (c + 1 < s.nc) {
    if (P.dt_bias) bias.y = P.dt_bias[s.c0 + c + 1];
    if (P.D) dskip.y = P.D[s.c0 + c + 1];
  }
  const u64 bias2 = pk2(bias.x, bias.y), skip2 = pk2(dskip.x, dskip.y);
  float2 sum_dD = zero2, sum_db = zero2;

  for (int tile = P.tiles - 1; tile >= 0; --tile) {
    const int t0 = tile * G::TL;
    __syncthreads();
    scan_stage<T, LT>(rx, P.x, P, s, t0);
    scan_stage<T, LT>(rdt, P.dt, P, s, t0);
    scan_stage<T, LT>(rdy, P.dy, P, s, t0);
    if (P.z.p) scan_stage<T, LT>(rz, P.z, P, s, t0);
    scan_stage_bc<T, LT>(Bs, P.Bm, P.b_sb, P.b_st, P.b_sg, P, s, t0, np2);
    scan_stage_bc<T, LT>(Cs, P.Cm, P.c_sb, P.c_st, P.c_sg, P, s, t0, np2);
    if (PACKED) {
      for (int i = threadIdx.x; i < G::TL; i += SCAN_THREADS) {
        first[i] = t0 + i < P.T ? __ldg(P.seq.start + t0 + i) : -1;
        last[i] = t0 + i < P.T ? __ldg(P.seq.end + t0 + i) : -1;
      }
    }
    {
      const float* ck = P.ckpt + (((long long)s.b * P.tiles + tile) * gridDim.x + blockIdx.x) * (N * G::CPB);
      for (int i = threadIdx.x; i < N * G::CPB; i += SCAN_THREADS) hst[i] = ck[i];
    }
    for (int i = threadIdx.x; i < 2 * N * G::TL; i += SCAN_THREADS) dBs[i] = 0.f;
    __syncthreads();

    u64 d[SCAN_K], u[SCAN_K], ds[SCAN_K], gb[SCAN_K], dd[SCAN_K], y[SCAN_K], sum;
    scan_inputs<T, LT>(P, rx, rdt, t0, tl, c, bias2, d, u, sum);
    ScanFlags f{};
    if (PACKED) f = scan_flags<LT>(first, last, tl);
#pragma unroll
    for (int j = 0; j < SCAN_K; ++j) {
      const int off = G::raw_off(tl * SCAN_K + j, c);
      float2 v = upk2(scan_pair<T>(rdy + off));
      if (P.z.p) {
        const float2 z = upk2(scan_pair<T>(rz + off));
        v.x *= siluf_(z.x);
        v.y *= siluf_(z.y);
      }
      ds[j] = pk2(v.x, v.y);
      gb[j] = dd[j] = y[j] = pk2(0.f, 0.f);
    }

    auto states = [&](auto reset) {
      constexpr bool RESET = decltype(reset)::value;
#pragma unroll 1
      for (int step = 0; step < steps; ++step) {
      const int n = step + warp < steps ? step + warp : step + warp - steps;
      if (n < N) {
        const u64 a2 = *reinterpret_cast<const u64*>(A2 + n * G::CPB + c);
        const u64 h_in = *reinterpret_cast<const u64*>(hst + n * G::CPB + c);
        const u64 g_in = *reinterpret_cast<const u64*>(gcar + n * G::CPB + c);
        float bv[SCAN_K], cv[SCAN_K];
        scan_row8(Bs + n * G::BCP, G::TL / 2, tl, bv);
        scan_row8(Cs + n * G::BCP, G::TL / 2, tl, cv);
        u64 a[SCAN_K], hh[SCAN_K];
#pragma unroll
        for (int j = 0; j < SCAN_K; ++j) {
          a[j] = ex2_2(mul2(d[j], a2));
          hh[j] = mul2(u[j], pk2(bv[j], bv[j]));
        }
        if (RESET && P.h0) {
#pragma unroll
          for (int j = 0; j < SCAN_K; ++j)
            if (f.first >> j & 1) {
              const float2 h = scan_state2(P.h0, first[tl * SCAN_K + j], P.E, N, c, s.nc, s.c0, n);
              hh[j] = fma2(a[j], pk2(h.x, h.y), hh[j]);
            }
        }
        const u64 p = ex2_2(mul2(sum, a2));
        // states of the tile
        u64 h = hh[0];
#pragma unroll
        for (int j = 1; j < SCAN_K; ++j) h = RESET && (f.first >> j & 1) ? hh[j] : fma2(a[j], h, hh[j]);
        if (tl == 0 && !(RESET && f.first)) h = fma2(p, h_in, h);
        scan_lanes<LT, RESET>(h, p, tl, f.up);
        h = scan_up<LT>(h, 1);
        if (tl == 0) h = h_in;
        const u64 h_first = h;
#pragma unroll
        for (int j = 0; j < SCAN_K; ++j) {
          h = RESET && (f.first >> j & 1) ? hh[j] : fma2(a[j], h, hh[j]);
          hh[j] = h;
        }
        // gradients of the states, from the tile's end
        u64 cg[SCAN_K];
#pragma unroll
        for (int j = 0; j < SCAN_K; ++j) cg[j] = mul2(ds[j], pk2(cv[j], cv[j]));
        if (PACKED && f.any_last && P.dht) {
#pragma unroll
          for (int j = 0; j < SCAN_K; ++j)
            if (f.last >> j & 1) {
              const float2 v = scan_state2(P.dht, last[tl * SCAN_K + j], P.E, N, c, s.nc, s.c0, n);
              cg[j] = add2(cg[j], pk2(v.x, v.y));
            }
        }
        u64 r = pk2(0.f, 0.f);
#pragma unroll
        for (int j = SCAN_K - 1; j >= 0; --j) {
          r = j == SCAN_K - 1 ? mul2(a[j], cg[j]) : mul2(a[j], add2(cg[j], r));
          if (RESET && (f.first >> j & 1)) r = pk2(0.f, 0.f);  // nothing passes a sequence's start
        }
        if (tl == LT - 1 && !(RESET && f.first)) r = fma2(p, g_in, r);
        scan_lanes_rev<LT, RESET>(r, p, tl, f.down);
        __syncwarp();  // every lane has read the carried gradient
        if (tl == 0) *reinterpret_cast<u64*>(gcar + n * G::CPB + c) = r;
        r = scan_down<LT>(r, 1);
        if (tl == LT - 1) r = g_in;
        u64 sA = LT == 32 ? dAs[n * DAW + threadIdx.x] : pk2(0.f, 0.f);
        const u64 an = mul2(a2, pk2(LN2, LN2));
        float dB[SCAN_K], dC[SCAN_K];
#pragma unroll
        for (int j = SCAN_K - 1; j >= 0; --j) {
          const u64 g = add2(cg[j], r);
          r = mul2(a[j], g);
          u64 q;
          if (RESET && (f.first >> j & 1)) {  // what reaches the initial state
            const int sq = first[tl * SCAN_K + j];
            if (P.dh0) scan_put_state2(P.dh0, sq, P.E, N, c, s.nc, s.c0, n, upk2(r));
            q = pk2(0.f, 0.f);
            if (P.h0) {
              const float2 h0 = scan_state2(P.h0, sq, P.E, N, c, s.nc, s.c0, n);
              q = mul2(r, pk2(h0.x, h0.y));
            }
            r = pk2(0.f, 0.f);
          } else {
            q = mul2(r, j ? hh[j - 1] : h_first);
          }
          dd[j] = fma2(q, an, dd[j]);
          sA = fma2(q, d[j], sA);
          gb[j] = fma2(g, pk2(bv[j], bv[j]), gb[j]);
          const float2 db = upk2(mul2(g, u[j])), dc = upk2(mul2(ds[j], hh[j]));
          dB[j] = db.x + db.y;
          dC[j] = dc.x + dc.y;
          if (P.z.p) y[j] = fma2(hh[j], pk2(cv[j], cv[j]), y[j]);
        }
        if (LT == 32) {
          dAs[n * DAW + threadIdx.x] = sA;
        } else {
          sA = scan_sum<LT>(sA);
          if (tl == 0) dAs[n * DAW + c / 2] = add2(dAs[n * DAW + c / 2], sA);
        }
        // over the warp's channel pairs, then onto the tile's sums
#pragma unroll
        for (int m = LT; m < 32; m <<= 1) {
#pragma unroll
          for (int j = 0; j < SCAN_K; ++j) {
            dB[j] += __shfl_xor_sync(0xffffffffu, dB[j], m);
            dC[j] += __shfl_xor_sync(0xffffffffu, dC[j], m);
          }
        }
        if (lane < LT) {
#pragma unroll
          for (int j = 0; j < SCAN_K; ++j) {
            const int o = n * G::TL + G::bc_off(tl * SCAN_K + j);
            dBs[o] += dB[j];
            dCs[o] += dC[j];
          }
        }
      }
      __syncthreads();
    }
    };
    if (PACKED && f.any_first) states(std::true_type{});
    else states(std::false_type{});

#pragma unroll
    for (int j = 0; j < SCAN_K; ++j) {
      const int t = tl * SCAN_K + j, off = G::raw_off(t, c);
      const u64 x2 = scan_pair<T>(rx + off);
      const float2 raw = upk2(add2(scan_pair<T>(rdt + off), bias2));
      if (P.z.p) {
        const float2 z = upk2(scan_pair<T>(rz + off)), dy = upk2(scan_pair<T>(rdy + off));
        const float2 v = upk2(fma2(skip2, x2, y[j]));
        scan_put<T>(rz + off, make_float2(dy.x * v.x * silu_slopef_(z.x), dy.y * v.y * silu_slopef_(z.y)));
      }
      const float2 px = upk2(mul2(ds[j], x2));
      sum_dD.x += px.x;
      sum_dD.y += px.y;
      float2 v = upk2(fma2(gb[j], x2, dd[j]));
      if (P.softplus) {
        v.x *= sigmoidf_(raw.x);
        v.y *= sigmoidf_(raw.y);
      }
      if (t0 + t >= P.T) v = zero2;
      sum_db.x += v.x;
      sum_db.y += v.y;
      scan_put<T>(rdt + off, v);
      scan_put<T>(rx + off, upk2(fma2(gb[j], d[j], mul2(ds[j], skip2))));
    }
    __syncthreads();
    scan_unstage<T, LT>(rx, P.dx, P, s, t0);
    scan_unstage<T, LT>(rdt, P.ddt, P, s, t0);
    if (P.z.p) scan_unstage<T, LT>(rz, P.dz, P, s, t0);
    float* part = P.bc_part + ((((long long)s.b * P.tiles + tile) * P.G + s.g) * P.blocks + s.blk) * (2 * N * G::TL);
    for (int i = threadIdx.x; i < 2 * N * G::TL; i += SCAN_THREADS) part[i] = dBs[i];
  }
  if (!PACKED && P.dh0)
    for (int i = threadIdx.x; i < N * G::CPB; i += SCAN_THREADS) {
      const int n = i / G::CPB, cc = i - n * G::CPB;
      if (cc < s.nc) P.dh0[((long long)s.b * P.E + s.c0 + cc) * N + n] = gcar[i];
    }
  // the row's dA, dD and d dt_bias: sums over the LT lanes of a channel pair
  float* e0 = P.e_part + ((long long)s.b * P.E + s.c0 + c) * (N + 2);
  float* e1 = e0 + N + 2;
  for (int n = 0; n < N; ++n) {
    const float2 v = upk2(LT == 32 ? scan_sum<LT>(dAs[n * DAW + threadIdx.x]) : dAs[n * DAW + c / 2]);
    if (tl == 0 && c < s.nc) e0[n] = v.x;
    if (tl == 0 && c + 1 < s.nc) e1[n] = v.y;
  }
  const float2 dD = upk2(scan_sum<LT>(pk2(sum_dD.x, sum_dD.y))), db = upk2(scan_sum<LT>(pk2(sum_db.x, sum_db.y)));
  if (tl == 0 && c < s.nc) { e0[N] = dD.x; e0[N + 1] = db.x; }
  if (tl == 0 && c + 1 < s.nc) { e1[N] = dD.y; e1[N + 1] = db.y; }
}

// dB and dC: the channel blocks' partial sums of a tile, summed in block order.
// One CTA column per (row, tile, group); thread i takes element i of [2][N][TL].
constexpr int SCAN_BC_THREADS = 256;
template <typename T, int LT>
__global__ void __launch_bounds__(SCAN_BC_THREADS) ssm_scan_bc_kernel(const float* part, int T_, int tiles, int Gr,
                                                                      int blocks, int N, T* dB, T* dC) {
  using G = ScanGeo<T, LT>;
  const int per = 2 * N * G::TL;
  const int i = blockIdx.y * SCAN_BC_THREADS + threadIdx.x;
  if (i >= per) return;
  const long long w = blockIdx.x;  // (row, tile, group)
  const float* p = part + w * blocks * (long long)per + i;
  float acc = 0.f;
#pragma unroll 8
  for (int k = 0; k < blocks; ++k) acc += p[(long long)k * per];
  const int half = i / (N * G::TL), rest = i - half * (N * G::TL), n = rest / G::TL, o = rest - n * G::TL;
  const int t = ((o & (G::TL / 2 - 1)) >> 2) * 8 + (o / (G::TL / 2)) * 4 + (o & 3);  // inverse of bc_off
  const int g = (int)(w % Gr);
  const long long bt = w / Gr;
  const int tile = (int)(bt % tiles);
  const long long b = bt / tiles;
  const int tok = tile * G::TL + t;
  if (tok < T_) (half ? dC : dB)[((b * T_ + tok) * Gr + g) * N + n] = io_from_f<T>(acc);
}

// One token for each of `rows` requests: the slot's state [E][N] is read, stepped
// and rewritten; every other input is a row.  Memory bound on the states.
// A thread owns 4 states of a channel (LP lanes per channel, y summed by shuffles) and
// walks the rows with its A in registers.
constexpr int STEP_THREADS = 256;
struct ScanStepParams {
  const void *x, *dt, *z, *Bm, *Cm;
  long long sx, sdt, sz, b_sb, b_sg, c_sb, c_sg;
  const float *A, *D, *dt_bias;
  float* state;
  const int* slots;
  int rows, E, N, G, pool;
  bool softplus;
  void* y;  // [rows][E]
  int* err;
};

template <typename T, int LP, bool VEC>
__global__ void __launch_bounds__(STEP_THREADS) ssm_scan_step_kernel(ScanStepParams P) {
  const long long idx = (long long)blockIdx.x * STEP_THREADS + threadIdx.x;
  const int e = (int)(idx / LP), n0 = (int)(idx % LP) * 4, N = P.N;
  const bool ok = e < P.E;  // (whole channels: the shuffles below stay inside one)
  const int ec = ok ? e : 0;
  float a[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = n0 + k < N ? __ldg(P.A + (long long)ec * N + n0 + k) * LOG2E : 0.f;
  const float D = P.D ? __ldg(P.D + ec) : 0.f, bias = P.dt_bias ? __ldg(P.dt_bias + ec) : 0.f;
  const int g = ec / (P.E / P.G);
  for (int r = blockIdx.y; r < P.rows; r += gridDim.y) {
    const int s = step_slot(P.slots, r, P.pool, P.err);
    float y = 0.f, x = 0.f;
    if (s >= 0 && ok) {
      float* st = P.state + ((long long)s * P.E + e) * N + n0;
      float h[4];
      if (VEC) {
        if (n0 < N) {
          const float4 v = *reinterpret_cast<const float4*>(st);
          h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = n0 + k < N ? st[k] : 0.f;
      }
      x = io_to_f(static_cast<const T*>(P.x)[r * P.sx + e]);
      float d = io_to_f(static_cast<const T*>(P.dt)[r * P.sdt + e]) + bias;
      if (P.softplus) d = softplusf_(d);
      const T* B = static_cast<const T*>(P.Bm) + r * P.b_sb + g * P.b_sg + n0;
      const T* C = static_cast<const T*>(P.Cm) + r * P.c_sb + g * P.c_sg + n0;
      const float u = d * x;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (n0 + k < N) {
          h[k] = fmaf(ex2(d * a[k]), h[k], u * io_to_f(B[k]));
          y = fmaf(h[k], io_to_f(C[k]), y);
        }
      }
      if (VEC) {
        if (n0 < N) *reinterpret_cast<float4*>(st) = make_float4(h[0], h[1], h[2], h[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n0 + k < N) st[k] = h[k];
      }
    }
#pragma unroll
    for (int m = LP / 2; m >= 1; m >>= 1) y += __shfl_xor_sync(0xffffffffu, y, m);
    if (ok && n0 == 0) {
      y = fmaf(D, x, y);
      if (P.z && s >= 0) y *= siluf_(io_to_f(static_cast<const T*>(P.z)[r * P.sz + e]));
      static_cast<T*>(P.y)[(long long)r * P.E + e] = io_from_f<T>(s >= 0 ? y : 0.f);
    }
  }
}

}  // namespace kda
