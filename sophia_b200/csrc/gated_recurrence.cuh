// Gated linear recurrence (one state per channel, gates per token and channel):
//   r = sigmoid(decay + decay_bias),  i = sigmoid(gate + gate_bias)
//   a = exp(A r)  (A <= 0),           b = sqrt(1 - a^2) i x
//   h[t] = a h[t-1] + b,              y = h silu(z)  (or h)
// forward, backward and single tokens.
//
// A CTA owns 64 channels of a row and goes through the tokens in order, a tile of
// 8 S tokens at a time: warp w has the w-th S tokens, a lane two channels.  A thread
// maps the state in front of its tokens to the one behind them, h -> P h + c;
// the maps of the warps in front, composed on the state that the tile starts
// from, give its own start.  So nothing is read twice and no state leaves the
// SM between tiles.  Few rows: a cluster of CTAs takes the tiles in turn and
// exchanges their maps through distributed shared memory, in the order of the
// tiles -- one pass over the data at any number of rows.
//
// 10 bytes an element (bf16, with z) against seven special functions (ex2 and rcp of three
// sigmoids, sqrt), which the SM makes at 16 a clock: 51 and 52 us per 4 x 4096 x 2048
// elements, so the decay's exponential is a polynomial on packed fp32 arithmetic, which
// also gives 1 - a^2 without cancellation.  (One special function less, rsqrt(w d d) w for
// sqrt(w) / d, took as long, and an input gate's d = 1 + e^44 and above overflowed it.)
//
// Measured at 4 x 4096 x 2048 bf16 with z: forward 108 us, backward 196 us (floors 51 and
// 92 us of bytes), 128 channel groups on 148 SMs in clusters of two; 32 x 512 x 2048, no
// cluster: 81 and 162 us; fp32, 2 x 4096 x 2048: 78 and 122 us (51 and 92).  What bounds
// them: latency at 128 registers and 3.3 warps a scheduler (47 and 49 % of the issue slots,
// 51 and 40 % of the special functions, 31 % of DRAM) and SMs left over; at that number the
// 16-bit backward spills 72 bytes a thread (48 without z at odd rows).  Tried: CTAs of 512
// threads, one an SM, without a cluster (111 and 195 us, but 273 against 233 for the forward
// of one row of 32768 tokens); 4 tokens a thread and three CTAs an SM (142 and 289 us); CTAs
// of 128 threads; a tile's gates ahead of the states of the one before (5 % slower).
//
// A run's decay P is the exponential of its tokens' summed logarithms: one rounding of 2^-24 where their product has one a
// token, which is what a state that remembers thousands of tokens would feel.
#pragma once

#include <cooperative_groups.h>
#include <cuda.h>  // CUtensorMap

#include <cfloat>
#include <cstring>

#include "ssm_common.cuh"

namespace kda {

namespace cg = cooperative_groups;

constexpr int REC_THREADS = 256;
constexpr int REC_WARPS = REC_THREADS / 32;
constexpr int REC_CTAS = 2;          // per SM: 128 registers a thread
constexpr int REC_CH = 64;           // channels of a CTA, two a lane
constexpr int REC_MAX_CLUSTER = 8;   // the portable limit
// Tokens of a thread: a tile of 8 S tokens of one tensor is 8 KB in every type.
template <typename T>
__host__ __device__ constexpr int rec_s() { return sizeof(T) == 2 ? 8 : 4; }
template <typename T>
__host__ __device__ constexpr int rec_tile() { return REC_WARPS * rec_s<T>(); }
// Rows of a staged tile: 64 channels; without 16-byte alignment 16-bit rows are copied in
// words from the word that holds their first element, which takes one more.
template <typename T, bool VEC>
__host__ __device__ constexpr int rec_pitch() { return REC_CH * (int)sizeof(T) + (!VEC && sizeof(T) == 2 ? 4 : 0); }
template <typename T, bool VEC>
__host__ __device__ constexpr int rec_tensor_bytes() { return rec_tile<T>() * rec_pitch<T, VEC>(); }
// Tiles in flight or in use: two CTAs of an SM share its 227 KB.
template <bool VEC>
__host__ __device__ constexpr int rec_fwd_stages() { return VEC ? 3 : 2; }
constexpr int REC_BWD_STAGES = 2;

// ---------------------------------------------------------------- arithmetic on two channels

__device__ __forceinline__ u64 ex2_2(u64 v) {
  const float2 f = upk2(v);
  return pk2(ex2(f.x), ex2(f.y));
}
__device__ __forceinline__ u64 rcp_2(u64 v) {
  const float2 f = upk2(v);
  return pk2(rcp(f.x), rcp(f.y));
}
__device__ __forceinline__ u64 all2(float v) { return pk2(v, v); }
__device__ __forceinline__ u64 sub2(u64 a, u64 b) {
  u64 r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The packed arithmetic's constants, as kernel parameters: operands from the constant bank or uniform registers;
// literals were moved into a pair of registers at every use (28 of then 141 instructions a pair of elements).
struct RecConst {
  u64 one, two, log2e, round, poly[6];
};
inline RecConst rec_const() {
  auto two = [](float v) {
    unsigned u;
    std::memcpy(&u, &v, 4);
    return (u64)u << 32 | u;
  };
  // a fit of (1 - 2^f) / f on [-1/2, 1/2], relative error 2.1e-8, highest power first; 1.5 2^23
  return {two(1.f), two(2.f), two(-LOG2E), two(12582912.f),
          {two(-0.000154035122f), two(-0.00133907353f), two(-0.00961823761f), two(-0.0555035733f), two(-0.240226492f),
           two(-0.693147182f)}};
}

// e = exp(-(v + bias)) from v and nb = -bias log2 e
__device__ __forceinline__ u64 rec_expneg(const RecConst& k, u64 v, u64 nb) { return ex2_2(fma2(v, k.log2e, nb)); }
__device__ __forceinline__ u64 rec_sig(const RecConst& k, u64 e) { return rcp_2(add2(e, k.one)); }
// v sigmoid(v)
__device__ __forceinline__ u64 rec_silu(const RecConst& k, u64 v) { return mul2(v, rec_sig(k, ex2_2(mul2(v, k.log2e)))); }
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// a = 2^l and w = 1 - a^2 for l <= 0, both with fp32 relative accuracy.  l = n + f, n the nearest whole
// number; q = 1 - 2^f is a polynomial times f, which keeps q accurate in relative terms next to 0;
// a = 2^n (1 - q), m = 1 - a = 2^n q + (1 - 2^n) cancels nowhere, w = m (2 - m).  CLAMP: l may be below -126; from
// -150 on, where fp32 has nothing below, a is 0 (2^-126 times a rate of 1e34 would count in the rate's gradient).
template <bool CLAMP>
__device__ __forceinline__ void rec_decay(const RecConst& k, u64 l, u64& a, u64& w) {
  const float2 lf = upk2(l);
  if (CLAMP) l = pk2(max_nan(lf.x, -126.f), max_nan(lf.y, -126.f));
  const u64 t = add2(l, k.round);  // the sum's low bits are n
  const u64 f = sub2(l, sub2(t, k.round));
  u64 p = fma2(k.poly[0], f, k.poly[1]);
#pragma unroll
  for (int i = 2; i < 6; ++i) p = fma2(p, f, k.poly[i]);
  const float2 tf = upk2(t);
  const u64 s = pk2(__int_as_float((__float_as_int(tf.x) << 23) + 0x3f800000),
                    __int_as_float((__float_as_int(tf.y) << 23) + 0x3f800000));
  const u64 q = mul2(p, f);
  a = mul2(s, sub2(k.one, q));
  if (CLAMP) {
    const float2 af = upk2(a);
    a = pk2(lf.x < -150.f ? 0.f : af.x, lf.y < -150.f ? 0.f : af.y);
  }
  const u64 m = fma2(s, q, sub2(k.one, s));
  w = mul2(m, sub2(k.two, m));
}
__device__ __forceinline__ u64 rec_sqrt(u64 w) {
  float2 f = upk2(w);
  asm("sqrt.approx.ftz.f32 %0, %0;" : "+f"(f.x));
  asm("sqrt.approx.ftz.f32 %0, %0;" : "+f"(f.y));
  return pk2(f.x, f.y);
}
// 1 / v, but 0 for v = 0: where nothing decays, nothing enters
__device__ __forceinline__ u64 rec_inverse(u64 v) {
  const float2 f = upk2(v);
  return pk2(f.x == 0.f ? 0.f : rcp(f.x), f.y == 0.f ? 0.f : rcp(f.y));
}

struct RecParams {
  RecConst k;
  CUtensorMap map[5];  // decay, x, gate, then forward z, backward dy and z: [B][T][E], boxes of a tile (16-byte pieces only)
  int* err;
  RowView x, decay, gate, z, dy;  // z.p null = no output gate
  const float *A, *decay_bias, *gate_bias, *h0, *dht;
  void *y, *dx, *ddecay, *dgate, *dz;
  float *ht, *dh0;
  float* ckpt;     // [B][tiles][E] states in front of every tile
  float* partial;  // [B * cluster][E][3]: dA, ddecay_bias, dgate_bias
  int B, T, E, tiles, cluster;
  SeqMap seq;
};

// ---------------------------------------------------------------- staged tiles

__device__ __forceinline__ void rec_bar_init(uint64_t* bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void rec_bar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
constexpr uint32_t REC_POLLS = 1u << 26;
__device__ __forceinline__ bool rec_bar_wait(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < REC_POLLS; ++i) {
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(smem_u32(bar)), "r"(parity)
                 : "memory");
    if (done) return true;
  }
  return false;
}
// Sixteen bytes to the same place of a CTA of the cluster, counted by its mbarrier at the place of `bar`.
__device__ __forceinline__ void rec_send(const void* slot, const void* bar, int cta, const float4& v) {
  uint32_t to, sig;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(slot)), "r"(cta));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(sig) : "r"(smem_u32(bar)), "r"(cta));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to),
               "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(sig)
               : "memory");
}
// A tile's box into shared memory; tokens and channels past the tensor arrive as zeros.  (ch is a multiple of 64.)
__device__ __forceinline__ void rec_tma(char* dst, const CUtensorMap* map, int ch, int t, int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(ch), "r"(t), "r"(b), "r"(smem_u32(bar))
      : "memory");
}

// Four bytes into shared memory, of which the first n are read and the others zero.
__device__ __forceinline__ void cp_async4n(void* smem, const void* gmem, int n) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(smem_u32(smem)), "l"(gmem), "r"(n) : "memory");
}

// One tensor's tile from `base` (the CTA's first channel of its row), in words.  Rows past T and channels past the
// width are not copied; what is computed from them is not used.  (A first or last word may be half inside.  Of the last
// one only the valid bytes are read; the first one's other half is the element in front of an odd address, which shares
// its aligned word.)
template <typename T>
__device__ __forceinline__ void rec_copy(char* dst, const T* base, long long st, int t0, int tokens, int nch) {
  constexpr int TILE = rec_tile<T>(), PITCH = rec_pitch<T, false>(), WORDS = PITCH / 4;
  for (int q = threadIdx.x; q < TILE * WORDS; q += REC_THREADS) {
    const int row = q / WORDS, word = q - row * WORDS;
    if (t0 + row >= tokens) break;
    const uintptr_t at = reinterpret_cast<uintptr_t>(base + (long long)(t0 + row) * st);
    const uintptr_t src = (at & ~uintptr_t(3)) + 4 * word, end = at + nch * sizeof(T);
    if (src < end)
      cp_async4n(dst + row * PITCH + word * 4, reinterpret_cast<const void*>(src), (int)min((unsigned long long)(end - src), 4ull));
  }
}

// A thread's two channels of a staged row: neighbours (VEC), or 32 apart.
template <typename T, bool VEC>
__device__ __forceinline__ u64 rec_get(const char* tile, int row, int odd) {
  const int lane = threadIdx.x & 31;
  const char* p = tile + row * rec_pitch<T, VEC>();
  if (VEC) {
    if (sizeof(T) == 4) return *reinterpret_cast<const u64*>(p + lane * 8);
    const IoVec<T, 2> v = *reinterpret_cast<const IoVec<T, 2>*>(p + lane * 4);
    return pk2(io_to_f(v.v[0]), io_to_f(v.v[1]));
  }
  const T* e = reinterpret_cast<const T*>(p) + odd + lane;
  return pk2(io_to_f(e[0]), io_to_f(e[32]));
}
// The same as it is stored, to be converted later.
template <typename T, bool VEC>
__device__ __forceinline__ IoVec<T, 2> rec_raw(const char* tile, int row, int odd) {
  const int lane = threadIdx.x & 31;
  const char* p = tile + row * rec_pitch<T, VEC>();
  if (VEC) return *reinterpret_cast<const IoVec<T, 2>*>(p + lane * 2 * sizeof(T));
  const T* e = reinterpret_cast<const T*>(p) + odd + lane;
  IoVec<T, 2> v;
  v.v[0] = e[0];
  v.v[1] = e[32];
  return v;
}
__device__ __forceinline__ int rec_lane_ch(bool vec, int k) {
  const int lane = threadIdx.x & 31;
  return vec ? 2 * lane + k : lane + 32 * k;
}
template <typename T, bool VEC>
__device__ __forceinline__ void rec_put(T* row, u64 v, int nch) {
  const float2 f = upk2(v);
  const int c0 = rec_lane_ch(VEC, 0), c1 = rec_lane_ch(VEC, 1);
  if (VEC) {  // nch is a multiple of 16 bytes' elements; a predicate, where a branch would cost three instructions
    if (sizeof(T) == 4) {
      asm volatile("{ .reg .pred p; setp.lt.s32 p, %2, %3; @p st.global.b64 [%0], %1; }" ::"l"(row + c0), "l"(v), "r"(c0),
                   "r"(nch)
                   : "memory");
    } else {
      IoVec<T, 2> o;
      o.v[0] = io_from_f<T>(f.x);
      o.v[1] = io_from_f<T>(f.y);
      asm volatile("{ .reg .pred p; setp.lt.s32 p, %2, %3; @p st.global.b32 [%0], %1; }" ::"l"(row + c0),
                   "r"(*reinterpret_cast<const uint32_t*>(&o)), "r"(c0), "r"(nch)
                   : "memory");
    }
  } else {
    if (c0 < nch) row[c0] = io_from_f<T>(f.x);
    if (c1 < nch) row[c1] = io_from_f<T>(f.y);
  }
}
// The rates: NaN for a positive one, whose normaliser is not real; -inf as the largest finite one (a closed gate times
// an infinity would be NaN).  And in log2 units.
__device__ __forceinline__ u64 rec_rates(u64 a) {
  auto rate = [](float v) { return v > 0.f ? __int_as_float(0x7fffffff) : max_nan(v, -FLT_MAX); };
  const float2 f = upk2(a);
  return pk2(rate(f.x), rate(f.y));
}
__device__ __forceinline__ u64 rec_log2_rates(u64 rates) {
  const float2 f = upk2(rates);
  return pk2(max_nan(f.x * LOG2E, -FLT_MAX), max_nan(f.y * LOG2E, -FLT_MAX));
}
// fp32 vectors over the channels
__device__ __forceinline__ u64 rec_vec(const float* p, bool vec, int nch, float none) {
  const int c0 = rec_lane_ch(vec, 0), c1 = rec_lane_ch(vec, 1);
  return pk2(p && c0 < nch ? p[c0] : none, p && c1 < nch ? p[c1] : none);
}
__device__ __forceinline__ void rec_put_vec(float* p, u64 v, bool vec, int nch) {
  const float2 f = upk2(v);
  const int c0 = rec_lane_ch(vec, 0), c1 = rec_lane_ch(vec, 1);
  if (c0 < nch) p[c0] = f.x;
  if (c1 < nch) p[c1] = f.y;
}

// Where a staged 16-bit row starts inside its first word (0 or 1 elements).
template <typename T, bool VEC>
__device__ __forceinline__ int rec_odd(const T* base, long long st, int t) {
  if (VEC || sizeof(T) == 4) return 0;
  return (int)((reinterpret_cast<uintptr_t>(base) >> 1) + (unsigned long long)t * (unsigned long long)st) & 1;
}

// The starts and ends of sequences among a warp's S tokens, as masks; lane j < 8 holds the sequence that starts at token
// j, lane 8 + j the one that ends there (S <= 8).
struct RecMarks {
  int mine;
  unsigned starts, ends;
};
template <int S>
__device__ __forceinline__ RecMarks rec_marks(const SeqMap& m, int t0) {
  RecMarks r{-1, 0u, 0u};
  if (!m.start) return r;
  const int lane = threadIdx.x & 31, t = t0 + (lane & 7);
  if (lane < 16 && (lane & 7) < S && t < m.T) r.mine = __ldg((lane < 8 ? m.start : m.end) + t);
  const unsigned b = __ballot_sync(0xffffffffu, r.mine >= 0);
  r.starts = b & 0xff;
  r.ends = (b >> 8) & 0xff;
  return r;
}

// Maps of the warps (and of the CTAs of a cluster): h -> P h + c per channel; `cut` (a bit per warp or CTA):
// a sequence starts (backward: ends) inside, so the result is c alone.  A map is P, P, c, c of a lane's channels.
__device__ __forceinline__ u64 rec_step_map(const float4& m, bool cut, u64 h) {
  const u64 c = pk2(m.z, m.w), n = fma2(pk2(m.x, m.y), h, c);
  return cut ? c : n;
}

// h through the maps from..to - 1 (REV: last first), one per 32 lanes; `marked`: P < 0 stands for a cut.
template <bool REV>
__device__ __forceinline__ void rec_fold(u64& h, const float4* maps, int from, int to, bool marked) {
  if (!marked) {
    for (int i = from; i < to; ++i) h = rec_step_map(maps[32 * (REV ? to - 1 - (i - from) : i)], false, h);
  } else {
    for (int i = from; i < to; ++i) {
      const float4 m = maps[32 * (REV ? to - 1 - (i - from) : i)];
      h = rec_step_map(m, m.x < 0.f, h);
    }
  }
}

// The whole CTA's map: the warps' maps in order (reverse: last first; `mask`: their cuts).  P < 0 stands for a
// cut inside (a product of decays is not negative).
template <typename Get>
__device__ __forceinline__ float4 rec_compose(Get get, unsigned mask, bool reverse) {
  u64 p = all2(1.f), c = 0ull;
#pragma unroll
  for (int k = 0; k < REC_WARPS; ++k) {
    const int w = reverse ? REC_WARPS - 1 - k : k;
    const float4 v = get(w);
    c = rec_step_map(v, mask >> w & 1, c);
    p = mul2(p, pk2(v.x, v.y));
  }
  const float2 pf = upk2(p), cf = upk2(c);
  return make_float4(mask ? -1.f : pf.x, mask ? -1.f : pf.y, cf.x, cf.y);
}

// ---------------------------------------------------------------- forward

struct RecTrue { static constexpr bool value = true; };
struct RecFalse { static constexpr bool value = false; };

struct RecFwdSmem {
  float4 maps[2][REC_WARPS][32];
  u64 carry[2][32];
  uint64_t full[3], peers[2];
  unsigned cuts[2][REC_WARPS];
};

__device__ __forceinline__ unsigned rec_cuts(const unsigned (&c)[REC_WARPS]) {
  unsigned m = 0;
#pragma unroll
  for (int w = 0; w < REC_WARPS; ++w) m |= c[w] ? 1u << w : 0u;
  return m;
}

template <typename T, bool VEC, bool Z>
__global__ void __launch_bounds__(REC_THREADS, REC_CTAS) rec_fwd_kernel(const __grid_constant__ RecParams P) {
  constexpr int S = rec_s<T>(), TILE = rec_tile<T>(), TB = rec_tensor_bytes<T, VEC>(), STAGES = rec_fwd_stages<VEC>();
  constexpr int STAGE_BYTES = (Z ? 4 : 3) * TB;
  extern __shared__ __align__(128) char stages[];
  __shared__ RecFwdSmem sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int nc = P.cluster, rank = nc > 1 ? (int)blockIdx.x % nc : 0;
  const int b = blockIdx.y, ch0 = (int)blockIdx.x / nc * REC_CH, nch = min(REC_CH, P.E - ch0);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const bool packed = P.seq.start != nullptr;
  const T* px = row_ptr<T>(P.x, b, 0) + ch0;
  const T* pd = row_ptr<T>(P.decay, b, 0) + ch0;
  const T* pg = row_ptr<T>(P.gate, b, 0) + ch0;
  const T* pz = Z ? row_ptr<T>(P.z, b, 0) + ch0 : nullptr;
  T* py = static_cast<T*>(P.y) + (long long)b * P.T * P.E + ch0;
  const int iters = (P.tiles + nc - 1) / nc;
  float4* peer_maps = reinterpret_cast<float4*>(stages + STAGES * STAGE_BYTES);  // [2][nc][32]: the cluster's
  bool alive = true;

  auto fetch = [&](int it) {
    char* s = stages + (it % STAGES) * STAGE_BYTES;
    const int t0 = (it * nc + rank) * TILE;
    if (VEC) {
      if (threadIdx.x == 0 && it < iters && alive) {
        uint64_t* bar = &sm.full[it % STAGES];
        rec_bar_expect(bar, STAGE_BYTES);
#pragma unroll
        for (int q = 0; q < (Z ? 4 : 3); ++q) rec_tma(s + q * TB, &P.map[q], ch0, t0, b, bar);
      }
    } else {
      if (it < iters) {
        rec_copy<T>(s, pd, P.decay.st, t0, P.T, nch);
        rec_copy<T>(s + TB, px, P.x.st, t0, P.T, nch);
        rec_copy<T>(s + 2 * TB, pg, P.gate.st, t0, P.T, nch);
        if (Z) rec_copy<T>(s + 3 * TB, pz, P.z.st, t0, P.T, nch);
      }
      cp_async_commit();
    }
  };
  if (threadIdx.x == 0) {
    for (int q = 0; q < STAGES; ++q) rec_bar_init(&sm.full[q]);
    rec_bar_init(&sm.peers[0]);
    rec_bar_init(&sm.peers[1]);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (nc > 1) cluster.sync();  // before any other CTA sends here
  else __syncthreads();
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) fetch(k);

  const RecConst& K = P.k;
  const u64 A2 = rec_log2_rates(rec_rates(rec_vec(P.A + ch0, VEC, nch, 0.f)));
  const u64 nd = mul2(rec_vec(P.decay_bias ? P.decay_bias + ch0 : nullptr, VEC, nch, 0.f), all2(-LOG2E));
  const u64 ng = mul2(rec_vec(P.gate_bias ? P.gate_bias + ch0 : nullptr, VEC, nch, 0.f), all2(-LOG2E));
  const bool steep = __any_sync(0xffffffffu, upk2(A2).x < -126.f || upk2(A2).y < -126.f);
  // the state in front of the cluster's first tile; then (one CTA) in shared memory, (several) composed by everyone
  u64 carry = packed ? 0ull : rec_vec(P.h0 ? P.h0 + (long long)b * P.E + ch0 : nullptr, VEC, nch, 0.f);
  auto h0_of = [&](const RecMarks& m, int j) {  // the state that the sequence starting at a warp's token j starts from
    const int q = __shfl_sync(0xffffffffu, m.mine, j);
    return rec_vec(P.h0 ? P.h0 + (long long)q * P.E + ch0 : nullptr, VEC, nch, 0.f);
  };

  int slot = 0, turn = 0;  // the tile's place among the stages, and the parity of its arrival
  for (int it = 0; it < iters; ++it, turn ^= slot == STAGES - 1, slot = slot == STAGES - 1 ? 0 : slot + 1) {
    const int tile = it * nc + rank, t0 = tile * TILE + warp * S, par = it & 1;
    const char* s = stages + slot * STAGE_BYTES;
    const int n = min(S, P.T - t0);  // tokens of this warp (may be <= 0)
    const RecMarks marks = rec_marks<S>(P.seq, t0);
    if (VEC) {
      if (alive) alive = rec_bar_wait(&sm.full[slot], turn);
    } else {
      cp_async_wait<STAGES - 2>();
      __syncthreads();
    }

    // gates, and the map of this warp's tokens
    const bool whole = n == S && !(marks.starts | marks.ends) && !steep;  // nothing special about them
    u64 a[S], bb[S];
    IoVec<T, 2> zr[S];
    u64 logs = 0ull, c = 0ull;
    auto gates = [&](auto all) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (!all.value && j >= n) break;
        const int row = warp * S + j, t = t0 + j;
        const u64 r = rec_sig(K, rec_expneg(K, rec_get<T, VEC>(s, row, rec_odd<T, VEC>(pd, P.decay.st, t)), nd));
        u64 w;
        const u64 l = mul2(A2, r);
        rec_decay<!all.value>(K, l, a[j], w);
        logs = add2(logs, l);
        const u64 i = rec_sig(K, rec_expneg(K, rec_get<T, VEC>(s + 2 * TB, row, rec_odd<T, VEC>(pg, P.gate.st, t)), ng));
        const u64 x = rec_get<T, VEC>(s + TB, row, rec_odd<T, VEC>(px, P.x.st, t));
        bb[j] = mul2(mul2(rec_sqrt(w), i), x);
        if (Z) zr[j] = rec_raw<T, VEC>(s + 3 * TB, row, rec_odd<T, VEC>(pz, P.z.st, t));
        if (!all.value && (marks.starts >> j & 1)) c = h0_of(marks, j);
        c = fma2(a[j], c, bb[j]);
      }
    };
    if (whole) gates(RecTrue{});
    else gates(RecFalse{});
    {
      u64 p, w;
      rec_decay<true>(K, logs, p, w);
      const float2 pf = upk2(p), cf = upk2(c);
      sm.maps[par][warp][lane] = make_float4(pf.x, pf.y, cf.x, cf.y);
      if (lane == 0) sm.cuts[par][warp] = marks.starts;
    }
    __syncthreads();  // the maps are there, and nobody reads the staged tile any more
    fetch(it + STAGES - 1);
    const unsigned cuts = packed ? rec_cuts(sm.cuts[par]) : 0u;

    u64 h;
    if (nc > 1) {  // the tiles of the cluster's other CTAs: their maps, in order
      if (warp == 0) {
        if (lane == 0) rec_bar_expect(&sm.peers[par], nc * 32 * (uint32_t)sizeof(float4));
        const float4 m = rec_compose([&](int w) { return sm.maps[par][w][lane]; }, cuts, false);
        for (int q = 0; q < nc; ++q) rec_send(&peer_maps[(par * nc + rank) * 32 + lane], &sm.peers[par], q, m);
      }
      if (alive) alive = rec_bar_wait(&sm.peers[par], (it >> 1) & 1);
      rec_fold<false>(carry, &peer_maps[par * nc * 32 + lane], 0, rank, packed);
      h = carry;
      rec_fold<false>(carry, &peer_maps[par * nc * 32 + lane], rank, nc, packed);
    } else {
      h = it > 0 ? sm.carry[par][lane] : carry;
    }
    if (P.ckpt && warp == 0 && tile < P.tiles)
      rec_put_vec(P.ckpt + ((long long)b * P.tiles + tile) * P.E + ch0, h, VEC, nch);
    if (!cuts) rec_fold<false>(h, &sm.maps[par][0][lane], 0, warp, false);
    else
      for (int w = 0; w < warp; ++w) h = rec_step_map(sm.maps[par][w][lane], cuts >> w & 1, h);

    // the states, and what leaves
    T* out = py + (long long)t0 * P.E;
    auto states = [&](auto all) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (!all.value && j >= n) break;
        if (!all.value && (marks.starts >> j & 1)) h = h0_of(marks, j);
        h = fma2(a[j], h, bb[j]);
        rec_put<T, VEC>(out + (long long)j * P.E, Z ? mul2(h, rec_silu(K, pk2(io_to_f(zr[j].v[0]), io_to_f(zr[j].v[1])))) : h, nch);
        if (!all.value && P.ht && (marks.ends >> j & 1)) {
          const int q = __shfl_sync(0xffffffffu, marks.mine, 8 + j);
          rec_put_vec(P.ht + (long long)q * P.E + ch0, h, VEC, nch);
        }
      }
    };
    if (whole) states(RecTrue{});
    else states(RecFalse{});
    if (warp == REC_WARPS - 1) {  // behind the tile's last token
      if (nc == 1) carry = h;
      sm.carry[par ^ 1][lane] = h;
    }
  }
  if (!packed && P.ht && rank == 0 && warp == REC_WARPS - 1)
    rec_put_vec(P.ht + (long long)b * P.E + ch0, carry, VEC, nch);
  if (!alive) atomicExch(P.err, 12);
  if (VEC) {
    if (!alive) {  // a copy or a map did not arrive: let what is in flight land (waiting again, as long)
      if (threadIdx.x == 0)
        for (int it = max(0, iters - STAGES); it < iters; ++it) rec_bar_wait(&sm.full[it % STAGES], (it / STAGES) & 1);
    }
  } else {
    cp_async_wait<0>();
  }
  if (nc > 1) cluster.sync();  // no CTA leaves while another may still write its maps here
}

// ---------------------------------------------------------------- backward

// With G[t] the gradient of h[t], from the last token to the first:
//   G[t] = dy silu(z) + a[t+1] G[t+1]   (at a sequence's last token: + dht instead)
//   dx = G n i,  dgate = G n x i (1 - i),  n = sqrt(1 - a^2);   dz = dy h silu'(z)
//   d(A r) = G (a h[t-1] - (a^2 / n) i x),  ddecay = d(A r) A r (1 - r),  dA = sum d(A r) r
// A warp's tokens map what comes from behind, U = a[t+1] G[t+1], to what they hand on: U -> P U + d with the same P
// as the states, so both directions meet in one exchange.  The states start from the tile's checkpoint.
struct RecBwdSmem {
  float4 maps[2][REC_WARPS][32];  // states: P, P, c, c
  float2 back[2][REC_WARPS][32];  // gradients: d, d (P as above)
  u64 carry[2][32];
  uint64_t full[REC_BWD_STAGES], peers[2];
  unsigned cuts[2][REC_WARPS], ends[2][REC_WARPS];
};

// Adds v to a compensated sum (s, c), which an infinity leaves infinite (inf - inf would make NaN of the error).
__device__ __forceinline__ void rec_add(u64& s, u64& c, u64 v) {
  const u64 y = sub2(v, c), t = add2(s, y);
  const float2 e = upk2(sub2(sub2(t, s), y)), f = upk2(t);
  c = pk2(fabsf(f.x) <= FLT_MAX ? e.x : 0.f, fabsf(f.y) <= FLT_MAX ? e.y : 0.f);
  s = t;
}

template <typename T, bool VEC, bool Z>
__global__ void __launch_bounds__(REC_THREADS, REC_CTAS) rec_bwd_kernel(const __grid_constant__ RecParams P) {
  constexpr int S = rec_s<T>(), TILE = rec_tile<T>(), TB = rec_tensor_bytes<T, VEC>(), STAGES = REC_BWD_STAGES;
  constexpr int STAGE_BYTES = (Z ? 5 : 4) * TB;
  extern __shared__ __align__(128) char stages[];
  __shared__ RecBwdSmem sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int nc = P.cluster, rank = nc > 1 ? (int)blockIdx.x % nc : 0;
  const int b = blockIdx.y, ch0 = (int)blockIdx.x / nc * REC_CH, nch = min(REC_CH, P.E - ch0);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const bool packed = P.seq.start != nullptr;
  const T* px = row_ptr<T>(P.x, b, 0) + ch0;
  const T* pd = row_ptr<T>(P.decay, b, 0) + ch0;
  const T* pg = row_ptr<T>(P.gate, b, 0) + ch0;
  const T* pz = Z ? row_ptr<T>(P.z, b, 0) + ch0 : nullptr;
  const T* pdy = row_ptr<T>(P.dy, b, 0) + ch0;
  const long long out0 = (long long)b * P.T * P.E + ch0;
  const int iters = (P.tiles + nc - 1) / nc;
  float4* peer_maps = reinterpret_cast<float4*>(stages + STAGES * STAGE_BYTES);  // [2][nc][32]: the cluster's

  bool alive = true;

  auto fetch = [&](int k) {  // the k-th tile from the end
    char* s = stages + (k % STAGES) * STAGE_BYTES;
    const int t0 = ((iters - 1 - k) * nc + rank) * TILE;
    if (VEC) {
      if (threadIdx.x == 0 && k < iters && alive) {
        uint64_t* bar = &sm.full[k % STAGES];
        rec_bar_expect(bar, STAGE_BYTES);
#pragma unroll
        for (int q = 0; q < (Z ? 5 : 4); ++q) rec_tma(s + q * TB, &P.map[q], ch0, t0, b, bar);
      }
    } else {
      if (k < iters) {
        rec_copy<T>(s, pd, P.decay.st, t0, P.T, nch);
        rec_copy<T>(s + TB, px, P.x.st, t0, P.T, nch);
        rec_copy<T>(s + 2 * TB, pg, P.gate.st, t0, P.T, nch);
        rec_copy<T>(s + 3 * TB, pdy, P.dy.st, t0, P.T, nch);
        if (Z) rec_copy<T>(s + 4 * TB, pz, P.z.st, t0, P.T, nch);
      }
      cp_async_commit();
    }
  };
  if (threadIdx.x == 0) {
    for (int q = 0; q < STAGES; ++q) rec_bar_init(&sm.full[q]);
    rec_bar_init(&sm.peers[0]);
    rec_bar_init(&sm.peers[1]);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (nc > 1) cluster.sync();  // before any other CTA sends here
  else __syncthreads();
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) fetch(k);

  const u64 A1 = rec_rates(rec_vec(P.A + ch0, VEC, nch, 0.f)), A2 = rec_log2_rates(A1);
  const u64 nd = mul2(rec_vec(P.decay_bias ? P.decay_bias + ch0 : nullptr, VEC, nch, 0.f), all2(-LOG2E));
  const u64 ng = mul2(rec_vec(P.gate_bias ? P.gate_bias + ch0 : nullptr, VEC, nch, 0.f), all2(-LOG2E));
  const bool steep = __any_sync(0xffffffffu, upk2(A2).x < -126.f || upk2(A2).y < -126.f);
  u64 carry = packed ? 0ull : rec_vec(P.dht ? P.dht + (long long)b * P.E + ch0 : nullptr, VEC, nch, 0.f);
  auto h0_of = [&](const RecMarks& m, int j) {
    const int q = __shfl_sync(0xffffffffu, m.mine, j);
    return rec_vec(P.h0 ? P.h0 + (long long)q * P.E + ch0 : nullptr, VEC, nch, 0.f);
  };
  auto dht_of = [&](const RecMarks& m, int j) {
    const int q = __shfl_sync(0xffffffffu, m.mine, 8 + j);
    return rec_vec(P.dht ? P.dht + (long long)q * P.E + ch0 : nullptr, VEC, nch, 0.f);
  };
  u64 sumA = 0ull, lowA = 0ull, sumD = 0ull, lowD = 0ull, sumG = 0ull, lowG = 0ull;

  for (int k = 0; k < iters; ++k) {
    const int tile = (iters - 1 - k) * nc + rank, t0 = tile * TILE + warp * S, par = k & 1;
    const char* s = stages + (k % STAGES) * STAGE_BYTES;
    u64 h = tile < P.tiles ? rec_vec(P.ckpt + ((long long)b * P.tiles + tile) * P.E + ch0, VEC, nch, 0.f) : 0ull;
    if (!VEC) cp_async_wait<STAGES - 2>();
    __syncthreads();  // nobody reads the tile before this one any more
    fetch(k + STAGES - 1);
    if (VEC && alive) alive = rec_bar_wait(&sm.full[k % STAGES], (k / STAGES) & 1);
    const int n = min(S, P.T - t0);
    const RecMarks marks = rec_marks<S>(P.seq, t0);

    auto get = [&](int which, const T* base, long long st, int j) {
      return rec_get<T, VEC>(s + which * TB, warp * S + j, rec_odd<T, VEC>(base, st, t0 + j));
    };
    const bool whole = n == S && !(marks.starts | marks.ends) && !steep;
    u64 a[S], hs[S], rr[S], ii[S], be[S];  // decay; b, then the state; the sigmoids; the normaliser
    {
      u64 p = all2(1.f), logs = 0ull, c = 0ull, d = 0ull;
      auto gates = [&](auto all) {
        bool open = true;  // no end among the tokens so far
#pragma unroll
        for (int j = 0; j < S; ++j) {
          if (!all.value && j >= n) break;
          rr[j] = rec_sig(P.k, rec_expneg(P.k, get(0, pd, P.decay.st, j), nd));
          u64 w;
          const u64 l = mul2(A2, rr[j]);
          rec_decay<!all.value>(P.k, l, a[j], w);
          logs = add2(logs, l);
          be[j] = rec_sqrt(w);
          ii[j] = rec_sig(P.k, rec_expneg(P.k, get(2, pg, P.gate.st, j), ng));
          hs[j] = mul2(mul2(be[j], ii[j]), get(1, px, P.x.st, j));
          u64 g = get(3, pdy, P.dy.st, j);
          if (Z) g = mul2(g, rec_silu(P.k, get(4, pz, P.z.st, j)));
          if (!all.value && (marks.starts >> j & 1)) c = h0_of(marks, j);
          c = fma2(a[j], c, hs[j]);
          p = mul2(p, a[j]);
          if (all.value || open) {
            if (!all.value && (marks.ends >> j & 1)) {
              g = add2(g, dht_of(marks, j));
              open = false;
            }
            d = fma2(p, g, d);
          }
        }
      };
      if (whole) gates(RecTrue{});
      else gates(RecFalse{});
      u64 w;
      rec_decay<true>(P.k, logs, p, w);
      const float2 pf = upk2(p), cf = upk2(c);
      sm.maps[par][warp][lane] = make_float4(pf.x, pf.y, cf.x, cf.y);
      sm.back[par][warp][lane] = upk2(d);
      if (lane == 0) {
        sm.cuts[par][warp] = marks.starts;
        sm.ends[par][warp] = marks.ends;
      }
    }
    __syncthreads();
    const unsigned cuts = packed ? rec_cuts(sm.cuts[par]) : 0u, ends = packed ? rec_cuts(sm.ends[par]) : 0u;
    auto back = [&](int w) {
      const float4 m = sm.maps[par][w][lane];
      const float2 d = sm.back[par][w][lane];
      return make_float4(m.x, m.y, d.x, d.y);
    };
    u64 U;
    if (nc > 1) {
      if (warp == 0) {
        if (lane == 0) rec_bar_expect(&sm.peers[par], nc * 32 * (uint32_t)sizeof(float4));
        const float4 m = rec_compose(back, ends, true);
        for (int q = 0; q < nc; ++q) rec_send(&peer_maps[(par * nc + rank) * 32 + lane], &sm.peers[par], q, m);
      }
      if (alive) alive = rec_bar_wait(&sm.peers[par], (k >> 1) & 1);
      rec_fold<true>(carry, &peer_maps[par * nc * 32 + lane], rank + 1, nc, packed);
      U = carry;
      rec_fold<true>(carry, &peer_maps[par * nc * 32 + lane], 0, rank + 1, packed);
    } else {
      U = k > 0 ? sm.carry[par][lane] : carry;
    }
    if (!(cuts | ends)) {
      for (int w = REC_WARPS - 1; w > warp; --w) U = rec_step_map(back(w), false, U);
      rec_fold<false>(h, &sm.maps[par][0][lane], 0, warp, false);
    } else {
      for (int w = REC_WARPS - 1; w > warp; --w) U = rec_step_map(back(w), ends >> w & 1, U);
      for (int w = 0; w < warp; ++w) h = rec_step_map(sm.maps[par][w][lane], cuts >> w & 1, h);
    }

    u64 tA = 0ull, tD = 0ull, tG = 0ull;
    const long long out = out0 + (long long)t0 * P.E;
    auto grads = [&](auto all) {
      const u64 h_in = h;
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (!all.value && j >= n) break;
        if (!all.value && (marks.starts >> j & 1)) h = h0_of(marks, j);
        h = fma2(a[j], h, hs[j]);
        hs[j] = h;
      }
#pragma unroll
      for (int j = S - 1; j >= 0; --j) {
        if (!all.value && j >= n) continue;
        const long long at = out + (long long)j * P.E;
        u64 prev = j > 0 ? hs[j > 0 ? j - 1 : 0] : h_in;
        if (!all.value && (marks.starts >> j & 1)) prev = h0_of(marks, j);
        u64 G = get(3, pdy, P.dy.st, j);
        if (Z) {  // silu' = s (1 + z (1 - s)) = s + z s (1 - s)
          const u64 z = get(4, pz, P.z.st, j), dyh = mul2(G, hs[j]);
          const u64 sg = rec_sig(P.k, ex2_2(mul2(z, P.k.log2e))), zs = mul2(z, sg);
          G = mul2(G, zs);
          rec_put<T, VEC>(static_cast<T*>(P.dz) + at, mul2(dyh, fma2(zs, sub2(P.k.one, sg), sg)), nch);
        }
        if (!all.value && (marks.ends >> j & 1)) U = dht_of(marks, j);
        G = add2(G, U);
        U = mul2(a[j], G);
        if (!all.value && (marks.starts >> j & 1) && P.dh0) {
          const int q = __shfl_sync(0xffffffffu, marks.mine, j);
          rec_put_vec(P.dh0 + (long long)q * P.E + ch0, U, VEC, nch);
        }
        const u64 ix = mul2(ii[j], get(1, px, P.x.st, j)), Gn = mul2(G, be[j]);
        rec_put<T, VEC>(static_cast<T*>(P.dx) + at, mul2(Gn, ii[j]), nch);
        const u64 dg = mul2(mul2(Gn, ix), sub2(P.k.one, ii[j]));
        rec_put<T, VEC>(static_cast<T*>(P.dgate) + at, dg, nch);
        tG = add2(tG, dg);
        // d(A r) r = G (a h' r - a^2 i x r / n): the small factors first, so that nothing overflows
        const u64 ar = mul2(a[j], rr[j]);
        const u64 dAr = mul2(G, sub2(mul2(ar, prev), mul2(mul2(ar, rec_inverse(be[j])), mul2(a[j], ix))));
        tA = add2(tA, dAr);
        const u64 dd = mul2(mul2(dAr, A1), sub2(P.k.one, rr[j]));
        rec_put<T, VEC>(static_cast<T*>(P.ddecay) + at, dd, nch);
        tD = add2(tD, dd);
      }
    };
    if (whole) grads(RecTrue{});
    else grads(RecFalse{});
    if (warp == 0) {  // in front of the tile's first token
      if (nc == 1) carry = U;
      sm.carry[par ^ 1][lane] = U;
    }
    rec_add(sumA, lowA, tA);
    rec_add(sumD, lowD, tD);
    rec_add(sumG, lowG, tG);
  }
  if (!packed && P.dh0 && rank == 0 && warp == 0) rec_put_vec(P.dh0 + (long long)b * P.E + ch0, carry, VEC, nch);
  if (!alive) atomicExch(P.err, 12);
  if (VEC) {
    if (!alive) {
      if (threadIdx.x == 0)
        for (int k = max(0, iters - STAGES); k < iters; ++k) rec_bar_wait(&sm.full[k % STAGES], (k / STAGES) & 1);
    }
  } else {
    cp_async_wait<0>();
  }
  __syncthreads();
  // the CTA's sums: the warps in order
  float* red = reinterpret_cast<float*>(stages);  // [warps][3][64]
  const u64 sums[3] = {sub2(sumA, lowA), sub2(sumD, lowD), sub2(sumG, lowG)};
#pragma unroll
  for (int q = 0; q < 3; ++q) rec_put_vec(red + (warp * 3 + q) * REC_CH, sums[q], VEC, REC_CH);
  __syncthreads();
  for (int i = threadIdx.x; i < 3 * REC_CH; i += REC_THREADS) {
    const int c = i / 3, q = i - 3 * c;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < REC_WARPS; ++w) t += red[(w * 3 + q) * REC_CH + c];
    if (c < nch) P.partial[(((long long)b * nc + rank) * P.E + ch0 + c) * 3 + q] = t;
  }
  if (nc > 1) cluster.sync();
}

// ---------------------------------------------------------------- single tokens

struct RecStepParams {
  RecConst k;
  const void *x, *decay, *gate, *z;
  long long sx, sd, sg, sz;
  const float *A, *decay_bias, *gate_bias;
  float* state;
  const int* slots;
  int rows, E, pool;
  void* y;
  int* err;
};

constexpr int REC_STEP_THREADS = 128;

// A thread has two neighbouring channels (VEC) or one, and strides over the rows: latency, not
// bandwidth, bounds every size that a decoding batch has.  The arithmetic is the prompt's, operation by operation.
template <typename T, bool VEC>
__global__ void __launch_bounds__(REC_STEP_THREADS) rec_step_kernel(const __grid_constant__ RecStepParams P) {
  constexpr int V = VEC ? 2 : 1;
  const int c = (blockIdx.x * REC_STEP_THREADS + threadIdx.x) * V;
  if (c >= P.E) return;
  auto vec = [&](const float* p) { return p ? pk2(__ldg(p + c), VEC ? __ldg(p + c + 1) : 0.f) : 0ull; };
  const u64 A2 = rec_log2_rates(rec_rates(vec(P.A)));
  const u64 nd = mul2(vec(P.decay_bias), all2(-LOG2E)), ng = mul2(vec(P.gate_bias), all2(-LOG2E));
  for (int r = blockIdx.y; r < P.rows; r += gridDim.y) {
    const int slot = step_slot(P.slots, r, P.pool, P.err);
    T* y = static_cast<T*>(P.y) + (long long)r * P.E + c;
    if (slot < 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) y[k] = io_from_f<T>(0.f);
      continue;
    }
    auto in = [&](const void* p, long long st) {
      float f[V];
      io_load<T, V>(static_cast<const T*>(p) + r * st + c, f);
      return pk2(f[0], f[V - 1]);
    };
    float* sp = P.state + (long long)slot * P.E + c;
    float hf[V];
    io_load<float, V>(sp, hf);
    const u64 rd = rec_sig(P.k, rec_expneg(P.k, in(P.decay, P.sd), nd)), gi = rec_sig(P.k, rec_expneg(P.k, in(P.gate, P.sg), ng));
    u64 a, w;
    rec_decay<true>(P.k, mul2(A2, rd), a, w);
    const u64 b = mul2(mul2(rec_sqrt(w), gi), in(P.x, P.sx));
    const u64 h = fma2(a, pk2(hf[0], hf[V - 1]), b);
    u64 o = h;
    if (P.z) {
      const u64 z = in(P.z, P.sz);
      o = mul2(h, mul2(z, rec_sig(P.k, ex2_2(mul2(z, P.k.log2e)))));
    }
    const float2 hn = upk2(h), on = upk2(o);
    const float h2[2] = {hn.x, hn.y}, o2[2] = {on.x, on.y};
    float hv[V], ov[V];
#pragma unroll
    for (int k = 0; k < V; ++k) hv[k] = h2[k], ov[k] = o2[k];
    io_store<float, V>(sp, hv);
    io_store<T, V>(y, ov);
  }
}

}  // namespace kda
