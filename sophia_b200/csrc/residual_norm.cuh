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
// 10 bytes an element forward and 16 backward when all is 16-bit; how rows are laid over
// threads, and what bounds that, stands at the two sorts of kernels: rows by bulk
// copies, and rows wherever they lie.
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
  long long params;   // floats from the ring's start to the parameters
  unsigned dense;     // bit per tensor (x, o, g, dv, dn): rows lie end to end
  int D, warps, lanes;  // a row's threads: warps of a group, or (one warp) that many lanes
  int parts;  // CTAs of the backward, set by its launch
  int* err;
  float eps;
};

// ---------------------------------------------------------------- rows

// Rows wherever they lie go element by element: four channels 32 apart, of which the first n are there, so that a warp's
// lanes have neighbours (with neighbours in a thread, a store touched four times the sectors: 98 and 320 us against 95 and
// 295, the two directions at 8192 x 2043).
template <typename T>
struct RnFour {
  T v[4];
  __device__ __forceinline__ void load(const T* q, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? q[32 * i] : io_from_f<T>(0.f);
  }
  __device__ __forceinline__ float get(int i) const { return io_to_f(v[i]); }
};
template <typename T>
__device__ __forceinline__ void rn_store(T* q, const float (&f)[4], int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) q[32 * i] = io_from_f<T>(f[i]);
}
__device__ __forceinline__ void rn_param(const float* p, int c, int n, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = i < n ? __ldg(p + c + 32 * i) : 0.f;
}
__device__ __forceinline__ int rn_there(int c, int D) { return min(4, max(0, (D - c + 31) >> 5)); }
// K = 2, eight channels a thread: four CTAs an SM forward and two backward, whose column sums then stay in registers;
// K = 4, rows above 2048 channels.  (8192 x 2043: 77 and 158 us, floors 36 and 56; with K = 4, its column sums in shared
// memory and three CTAs an SM launched where two fitted, 95 and 295.)
__host__ __device__ constexpr int rn_plain_threads(int k) { return k == 2 ? 256 : 512; }
template <typename T>
__device__ __forceinline__ const T* rn_row(const RowView& r, long long row, int T_) {
  if (T_ == 0) return static_cast<const T*>(r.p) + row * r.st;
  const long long b = row / T_;
  return static_cast<const T*>(r.p) + b * r.sb + (row - b * T_) * r.st;
}

// Sums over the `warps` warps of a row's group, the same in every thread.  `part` is another one than at the sum before, so
// that one barrier is enough.
template <int N>
__device__ __forceinline__ void rn_sum(float (&a)[N], float (*part)[RN_MAX_WARPS], int group, int warps) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] += __shfl_xor_sync(0xffffffffu, a[i], m);
  if (warps == 1) return;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) part[i][threadIdx.x >> 5] = a[i];
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) {
    a[i] = 0.f;
    for (int w = 0; w < warps; ++w) a[i] += part[i][group * warps + w];
  }
}

// ---------------------------------------------------------------- dropout

__device__ __forceinline__ uint4 philox(uint4 c, unsigned k0, unsigned k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    // (halves apart: as 64-bit products, 154 us against 90 of the forward of 16384 x 1536)
    const unsigned l0 = 0xD2511F53u * c.x, h0 = __umulhi(0xD2511F53u, c.x);
    const unsigned l1 = 0xCD9E8D57u * c.z, h1 = __umulhi(0xCD9E8D57u, c.z);
    c = make_uint4(h1 ^ c.y ^ k0, l1, h0 ^ c.w ^ k1, l0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}
// Bit i: channel c + 32 i is kept.  c - lane is a multiple of 128; the whole warp calls.  A lane draws the four words of
// the lane % 4-th 32 channels' group lane / 4, and the warp's votes on them give every lane its own.
__device__ __forceinline__ unsigned rn_kept(const RnParams& P, unsigned k0, unsigned k1, long long row, int c) {
  const int lane = threadIdx.x & 31, first = c - lane;
  const uint4 r = philox(make_uint4((unsigned)first / 4 + 8 * (lane & 3) + lane / 4, (unsigned)row, (unsigned)(row >> 32), P.offset),
                         k0, k1);
  const unsigned b0 = __ballot_sync(0xffffffffu, r.x >= P.drop), b1 = __ballot_sync(0xffffffffu, r.y >= P.drop);
  const unsigned b2 = __ballot_sync(0xffffffffu, r.z >= P.drop), b3 = __ballot_sync(0xffffffffu, r.w >= P.drop);
  const unsigned b = lane & 2 ? (lane & 1 ? b3 : b2) : (lane & 1 ? b1 : b0);
  return P.drop_all ? 0u : b >> (lane & ~3) & 15u;
}

// ---------------------------------------------------------------- forward, rows wherever they lie

// A group of warps has a row, in registers between its two reductions.  Instructions bound it: 116 an element at 75 % of
// the issue slots (predicates and addresses of single elements), DRAM at 32 %; the backward 163 at 55 %.
template <typename TX, typename TO, int K>
__global__ void __launch_bounds__(rn_plain_threads(K), K == 2 ? 4 : 1) rn_fwd_kernel(const __grid_constant__ RnParams P) {
  __shared__ float part[2][1][RN_MAX_WARPS];
  int flip = 0;
  const int warps = P.warps, group = (threadIdx.x >> 5) / warps, groups = (blockDim.x >> 5) / warps;
  const int me = threadIdx.x - group * warps * 32, stride = warps * 128, c0 = me / 32 * 128 + me % 32;
  const unsigned long long seed = P.seed_ptr ? (unsigned long long)*P.seed_ptr : P.seed;
  const unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  const float inv = 1.f / P.D;
  for (long long row = (long long)blockIdx.x * groups + group; row < P.rows; row += (long long)gridDim.x * groups) {
    const TX* px = rn_row<TX>(P.x, row, P.T);
    const TO* po = rn_row<TO>(P.o, row, P.T);
    const TO* pg = P.g.p ? rn_row<TO>(P.g, row, P.T) : nullptr;
    RnFour<TO> o[K], g[K];
    RnFour<TX> x[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = c0 + k * stride, n4 = rn_there(c, P.D);
      o[k].load(po + c, n4);
      x[k].load(px + c, n4);
      if (pg) g[k].load(pg + c, n4);
    }
    float rb = 1.f;
    if (P.wb) {
      float ss[1] = {0.f};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) ss[0] = fmaf(o[k].get(i), o[k].get(i), ss[0]);
      rn_sum(ss, part[flip ^= 1], group, warps);
      rb = rsqrtf(fmaf(ss[0], inv, P.eps));
    }
    float v[K][4], ss[1] = {0.f};
    TX* pv = static_cast<TX*>(P.v) + row * P.D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = c0 + k * stride, n4 = rn_there(c, P.D);
      const unsigned kept = P.dropout ? rn_kept(P, k0, k1, row, c) : 15u;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k][i] = 0.f;
      if (n4 > 0) {
        float f[4], u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = o[k].get(i);
        if (P.wb) {
          rn_param(P.wb, c, n4, f);
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] *= rb * f[i];
        }
        if (pg)
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] *= sigmoidf_(g[k].get(i));
        if (P.dropout)
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] = kept >> i & 1 ? P.keep_scale * u[i] : 0.f;
        if (P.scale) {
          rn_param(P.scale, c, n4, f);
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] *= f[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[k][i] = x[k].get(i) + u[i];
          ss[0] = fmaf(v[k][i], v[k][i], ss[0]);
        }
        rn_store(pv + c, v[k], n4);
      }
    }
    float r = 0.f;
    if (P.w) {
      rn_sum(ss, part[flip ^= 1], group, warps);
      r = rsqrtf(fmaf(ss[0], inv, P.eps));
      TO* pn = static_cast<TO*>(P.n) + row * P.D;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = c0 + k * stride, n4 = rn_there(c, P.D);
        if (n4 > 0) {
          float f[4];
          rn_param(P.w, c, n4, f);
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] *= v[k][i] * r;
          rn_store(pn + c, f, n4);
        }
      }
    }
    if (P.rstd && me == 0) {
      P.rstd[2 * row] = rb;
      P.rstd[2 * row + 1] = r;
    }
  }
}

// ---------------------------------------------------------------- rows by bulk copies

// Aligned rows come into a ring of stages in shared memory by bulk copies, so that the next rows are on their way
// while one is worked on.  A group of W warps owns a row at a time (NARROW rows, up to 256 channels: `lanes` lanes of a
// single warp, which has 32 / lanes rows at once); rows that lie end to end are one copy (small copies cost the copy
// engine as much as large ones), so a stage of short rows holds several.  A thread has the same channels in every
// row -- 16 to 32 forward, 16 backward, whose sums over rows stay in its registers, 8 of NARROW rows -- and computes in
// packed fp32 arithmetic; the parameters lie in shared memory.
// What a row costs beside its arithmetic -- waiting, barriers, sums over warps, addresses -- is what bounds these
// kernels, so the parts that a call has are known to the compiler as far as they change the loops (FULL: a row fills its
// threads; GATE; DROP).  Measured at 4 x 4096 x 1536, bf16 with an fp32 stream, norms on both sides, gate and dropout:
// forward 72 us and backward 128 us (75 and 66 % of the copy bandwidth); 2 x 4096 x 4096 bf16 without gate and dropout:
// 51 and 104 us (80 and 59 %).
// What each switch brings, known to the compiler and decided in the kernel (between events, forward + backward): GATE at
// 16384 x 1536 67 + 110 and 66 + 130 us, with dropout 71 + 134 and 71 + 188; DROP there 71 + 134 and 69 + 138, without
// dropout 67 + 110 and 65 + 122; FULL at 8192 x 4096 55 + 109 and 53 + 114, with gate and dropout 74 + 157 and 79 + 159,
// at 200 x 1536 13 + 28 and 14 + 30, but at 16384 x 1536 with gate and dropout 71 + 134 and 65 + 126: its rows of 24
// channels a thread would be better off without.
// Tried: a warp of its own for the copies (17 warps: 96 registers, spills); parameters from global memory; 8 channels a
// thread (forward 124 us); 16 channels of narrow rows (backward of 32768 x 256 88 us against 69).
constexpr int RN_MAX_STAGES = 4;
constexpr int RN_MAX_GROUPS = 16;

__device__ __forceinline__ void rn_bar_init(uint64_t* bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void rn_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void rn_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
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

// A tensor of the ring, held by one lane of a group's first warp: the lanes issue a stage's copies side by side (one after
// the other, with the addresses of five tensors, they held the group up for 1100 to 1800 cycles a row).
struct RnSource {
  const char* p;
  long long sb, st;    // bytes
  uint32_t row, off;   // bytes of a row, of the tensors in front of it in a stage (per row)
  bool dense, any;     // rows lie end to end; there is such a tensor for this lane
};
__device__ __forceinline__ RnSource rn_source(const RowView& r, uint32_t esz, uint32_t off, bool dense, int D) {
  return {static_cast<const char*>(r.p), r.sb * (long long)esz, r.st * (long long)esz, D * esz, off, dense, r.p != nullptr};
}
// n rows from row0 on to the stage at `at`, which has room for `rows`.
__device__ __forceinline__ void rn_copy(const RnSource& t, uint32_t at, int rows, long long row0, int n, int T, uint64_t* bar) {
  const uint32_t dst = at + rows * t.off;
  auto src = [&](long long row) {
    if (T == 0) return t.p + row * t.st;
    const long long b = row / T;
    return t.p + b * t.sb + (row - b * T) * t.st;
  };
  if (!t.any) return;
  if (t.dense) {
    rn_bulk(dst, src(row0), n * t.row, bar);
  } else {
    for (int i = 0; i < n; ++i) rn_bulk(dst + i * t.row, src(row0 + i), t.row, bar);
  }
}
// What a CTA shares: the sums' places (two for each group: a sum's may be written while the last one is read; a group's
// warps take whole fours of them) and the stages' arrivals.
constexpr int RN_PARTS = 32;
template <int N>
struct RnShared {
  float part[2][N][RN_PARTS];
  uint64_t full[RN_MAX_GROUPS][RN_MAX_STAGES];
};
// The parameters in shared memory [2][D]: w, and w_b scale, the only form in which a row needs those two.
__device__ __forceinline__ void rn_params(const RnParams& P, float* dst) {
  const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
  for (int c = threadIdx.x * 4; c < P.D; c += blockDim.x * 4) {
    const float4 b = P.wb ? __ldg(reinterpret_cast<const float4*>(P.wb + c)) : one;
    const float4 s = P.scale ? __ldg(reinterpret_cast<const float4*>(P.scale + c)) : one;
    if (P.w) *reinterpret_cast<float4*>(dst + c) = __ldg(reinterpret_cast<const float4*>(P.w + c));
    *reinterpret_cast<float4*>(dst + P.D + c) = make_float4(b.x * s.x, b.y * s.y, b.z * s.z, b.w * s.w);
  }
}

// A group's walk through its rows: where it and its thread stand, and its stages.
template <typename T, bool NARROW, int N>
struct RnGroup {
  int group, warps, lanes;
  int per, sub, me;   // rows that it works on at once, which of them, and the thread's number in that row
  int stride;         // channels between a thread's pieces
  int rows, batch;    // of a stage: rows, and how often `per`
  int first, step;    // its first row, and the rows between its stages
  int total;          // rows of the call
  bool leads, alive;  // the first warp; no wait has run out
  uint32_t base, stage_bytes, row_bytes;
  uint64_t* full;
  float (*part)[N][RN_PARTS];
  int place;  // its first of the sums' places
  int slot, turn, stages, flip;
  int refill, spare;  // the first row of the stage to be filled again once everyone has read it (or total), and that stage
  int T_;
  RnSource mine;

  __device__ __forceinline__ RnGroup(const RnParams& P, RnShared<N>& sh, uint32_t ring, uint32_t bytes_a_row) {
    constexpr int V = 16 / sizeof(T);
    warps = NARROW ? 1 : P.warps;
    lanes = P.lanes;
    const int groups = (int)(blockDim.x >> 5) / warps;
    group = (int)(threadIdx.x >> 5) / warps;
    const int in = threadIdx.x - group * warps * 32;
    per = NARROW ? 32 / lanes : 1;
    sub = NARROW ? in / lanes : 0;
    me = NARROW ? in % lanes : in;
    stride = (NARROW ? lanes : warps * 32) * V;
    batch = P.batch;
    rows = per * batch;
    total = (int)P.rows;
    first = ((int)blockIdx.x * groups + group) * rows;
    step = (int)gridDim.x * groups * rows;
    leads = in < 32;
    alive = true;
    row_bytes = bytes_a_row;
    stage_bytes = rows * row_bytes;
    stages = P.stages;
    base = ring + group * stages * stage_bytes;
    full = sh.full[group];
    part = sh.part;
    place = group * ((warps + 3) & ~3);
    slot = turn = flip = spare = 0;
    refill = total;
    T_ = P.T;
    mine = RnSource{};
    if (in == 0)
      for (int q = 0; q < stages; ++q) rn_bar_init(&full[q]);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = threadIdx.x; i < 2 * N * RN_PARTS; i += blockDim.x) (&sh.part[0][0][0])[i] = 0.f;
  }
  __device__ __forceinline__ void sync() const {
    if (warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
  }
  __device__ __forceinline__ void fetch(int row0, int s) {  // (the first warp)
    if (row0 >= total || !alive) return;
    const int n = min(rows, total - row0);
    if ((threadIdx.x & 31) == 0) rn_expect(&full[s], n * row_bytes);
    rn_copy(mine, base + s * stage_bytes, rows, row0, n, T_, &full[s]);
  }
  __device__ __forceinline__ void start() {
    if (leads)
      for (int q = 0; q < stages; ++q)
        if (first + (long long)q * step < total) fetch(first + q * step, q);
  }
  // Behind a barrier of the group in a row, everyone has read the stage before the row's own.
  __device__ __forceinline__ void again() {
    if (leads && refill < total) fetch(refill, spare);
    refill = total;
  }
  __device__ __forceinline__ void wait() {
    if (alive) alive = rn_wait(&full[slot], turn);
  }
  __device__ __forceinline__ void next(int row0) {
    spare = slot;
    refill = (long long)row0 + (long long)stages * step < total ? row0 + stages * step : total;
    if (stages == 1) {  // nothing on its way meanwhile
      sync();
      again();
    }
    if (++slot == stages) slot = 0, turn ^= 1;
  }
  __device__ __forceinline__ void finish(int* err) {
    if (alive) return;  // a copy did not arrive: report it, and let what is in flight land (waiting again, as long)
    atomicExch(err, 12);
    if (leads)
      for (int q = 0; q < stages; ++q) rn_wait(&full[q], q < slot ? turn ^ 1 : turn);
  }
  // The sums over a row's threads, the same in all of them.
  __device__ __forceinline__ void sum(float (&a)[N]) {
    if (NARROW) {
      for (int m = lanes >> 1; m >= 1; m >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] += __shfl_xor_sync(0xffffffffu, a[i], m);
      __syncwarp();
    } else {
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] += __shfl_xor_sync(0xffffffffu, a[i], m);
      if (warps > 1) {
        float (*p)[RN_PARTS] = part[flip];
        flip ^= 1;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
          for (int i = 0; i < N; ++i) p[i][place + (threadIdx.x >> 5) - group * warps] = a[i];
        sync();
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float4* q = reinterpret_cast<const float4*>(p[i] + place);
          float4 f = q[0];
          float t = (f.x + f.y) + (f.z + f.w);
          for (int w = 4; w < warps; w += 4) {
            f = q[w / 4];
            t += (f.x + f.y) + (f.z + f.w);
          }
          a[i] = t;
        }
      } else {
        __syncwarp();
      }
    }
    again();
  }
};

// V channels as pairs, from and to pieces of 16 bytes.
__device__ __forceinline__ u64 rn_pair(bf16, uint32_t u) { return pk2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ u64 rn_pair(f16, uint32_t u) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  return pk2(f.x, f.y);
}
__device__ __forceinline__ uint32_t rn_word(bf16, u64 v) {
  const float2 f = upk2(v);
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t rn_word(f16, u64 v) {
  const float2 f = upk2(v);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T, int V>
__device__ __forceinline__ void rn_take(uint32_t at, u64 (&f)[V / 2]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(f[2 * i]), "=l"(f[2 * i + 1]) : "r"(at + 16 * i));
  } else {
    uint32_t r[4];
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = rn_pair(T(), r[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void rn_put(T* q, const u64 (&f)[V / 2]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) reinterpret_cast<ulonglong2*>(q)[i] = make_ulonglong2(f[2 * i], f[2 * i + 1]);
  } else {
    *reinterpret_cast<uint4*>(q) = make_uint4(rn_word(T(), f[0]), rn_word(T(), f[1]), rn_word(T(), f[2]), rn_word(T(), f[3]));
  }
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


template <typename TX, typename TO, int K, bool NARROW, bool FULL, bool GATE, bool DROP>
__global__ void __launch_bounds__(RN_MAX_WARPS * 32, 1) rn_fwd_ring_kernel(const __grid_constant__ RnParams P) {
  constexpr int V = 16 / sizeof(TO), H = V / 2;
  extern __shared__ __align__(128) char ring[];  // the groups' stages, then the parameters [2][D]
  __shared__ __align__(16) RnShared<1> sh;
  const int D = P.D;
  const uint32_t xb = D * sizeof(TX), ob = D * sizeof(TO);
  RnGroup<TO, NARROW, 1> a(P, sh, smem_u32(ring), xb + (GATE ? 2 : 1) * ob);
  {
    const int lane = threadIdx.x & 31;
    if (lane == 0) a.mine = rn_source(P.x, sizeof(TX), 0, P.dense & 1, D);
    if (lane == 1) a.mine = rn_source(P.o, sizeof(TO), xb, P.dense >> 1 & 1, D);
    if (GATE && lane == 2) a.mine = rn_source(P.g, sizeof(TO), xb + ob, P.dense >> 2 & 1, D);
  }
  float* params = reinterpret_cast<float*>(ring) + P.params;
  __syncthreads();
  a.start();
  rn_params(P, params);
  __syncthreads();
  const bool has_w = P.w != nullptr, has_wb = P.wb != nullptr, has_ws = P.wb || P.scale, keeps = P.rstd && a.me == 0;
  unsigned long long seed = 0;
  if (DROP) seed = P.seed_ptr ? (unsigned long long)*P.seed_ptr : P.seed;
  const unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  const float inv = 1.f / D, eps = P.eps, keep = DROP ? P.keep_scale : 1.f;
  bool mine[K];  // the thread's pieces that there are
#pragma unroll
  for (int k = 0; k < K; ++k) mine[k] = FULL || a.me * V + k * a.stride < D;
  const uint32_t pw = smem_u32(params) + a.me * V * 4, pws = pw + 4 * D, kp = a.stride * 4;
  const uint32_t at_x = a.sub * xb + a.me * (V * (uint32_t)sizeof(TX)), at_o = a.rows * xb + a.sub * ob + a.me * 16;
  const uint32_t kx = a.stride * (uint32_t)sizeof(TX), ko = a.stride * (uint32_t)sizeof(TO), at_g = a.rows * ob;
  for (int row0 = a.first; row0 < a.total; row0 += a.step) {
    a.wait();
    uint32_t px = a.base + a.slot * a.stage_bytes + at_x, po = a.base + a.slot * a.stage_bytes + at_o;
    int row = row0 + a.sub;
    for (int j = 0; j < a.batch && row - a.sub < a.total; ++j, row += a.per, px += a.per * xb, po += a.per * ob) {
      const bool here = !NARROW || row < a.total;
      const long long out = (long long)row * D + a.me * V;
      u64 v[K][H], ss = 0ull;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (mine[k] && here) rn_take<TO, V>(po + k * ko, v[k]);
        else
#pragma unroll
          for (int i = 0; i < H; ++i) v[k][i] = 0ull;
      }
      float rb = 1.f, t[1];
      if (has_wb) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < H; ++i) ss = fma2(v[k][i], v[k][i], ss);
        t[0] = rn_hsum(ss);
        a.sum(t);
        rb = rsqrtf(fmaf(t[0], inv, eps));
        ss = 0ull;
      }
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (mine[k] && here) {
          u64 f[H];
          if (has_ws) {
            rn_take<float, V>(pws + k * kp, f);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], mul2(f[i], rn_all(rb)));
          }
          if (GATE) {
            rn_take<TO, V>(po + at_g + k * ko, f);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], rn_sigmoid(f[i]));
          }
          if (DROP) {
            const unsigned bits = rn_bits<V>(P, k0, k1, row, a.me * V + k * a.stride);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = rn_mask(mul2(v[k][i], rn_all(keep)), bits, i);
          }
          rn_take<TX, V>(px + k * kx, f);
#pragma unroll
          for (int i = 0; i < H; ++i) {
            v[k][i] = add2(v[k][i], f[i]);
            ss = fma2(v[k][i], v[k][i], ss);
          }
          rn_put<TX, V>(static_cast<TX*>(P.v) + out + k * a.stride, v[k]);
        }
      float r = 0.f;
      if (has_w) {
        t[0] = rn_hsum(ss);
        a.sum(t);
        r = rsqrtf(fmaf(t[0], inv, eps));
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (mine[k] && here) {
            u64 f[H];
            rn_take<float, V>(pw + k * kp, f);
#pragma unroll
            for (int i = 0; i < H; ++i) v[k][i] = mul2(v[k][i], mul2(f[i], rn_all(r)));
            rn_put<TO, V>(static_cast<TO*>(P.n) + out + k * a.stride, v[k]);
          }
      }
      if (keeps && here) *reinterpret_cast<float2*>(P.rstd + 2LL * row) = make_float2(rb, r);
      if (!has_w && !has_wb) {
        a.sync();
        a.again();
      }
    }
    a.next(row0);
  }
  a.finish(P.err);
}

// One round of sums a row: with t = scale m s u (what the stream got from the branch), the sum that the branch's norm
// needs is that of t dv', and dv' = dv + r (tw - v r^2 S1 / D) with tw = dn w, S1 = sum tw v: sum t dv' =
// sum t (dv + r tw) - r^3 S1 / D sum t v, and do = r_b (du w_b - o r_b / D sum t dv').  And one column sum serves two
// parameters: with Q = sum over the rows of m dv' s o r_b, dw_b = scale Q and dscale = w_b Q.
template <typename TX, typename TO, bool NARROW, bool FULL, bool GATE, bool DROP>
__global__ void __launch_bounds__(RN_MAX_WARPS * 32, 1) rn_bwd_ring_kernel(const __grid_constant__ RnParams P) {
  constexpr int V = 16 / sizeof(TO), H = V / 2, K = (NARROW ? 8 : 16) / V;
  extern __shared__ __align__(128) char ring[];  // the groups' stages, then the parameters [2][D], at the end the column sums
  __shared__ __align__(16) RnShared<3> sh;
  const int D = P.D;
  const bool has_dv = P.dv.p != nullptr, has_dn = P.dn.p != nullptr, has_wb = P.wb != nullptr;
  const uint32_t xb = D * sizeof(TX), ob = D * sizeof(TO);
  const uint32_t off_g = xb + ob, off_dv = off_g + (GATE ? ob : 0), off_dn = off_dv + (has_dv ? xb : 0);
  RnGroup<TO, NARROW, 3> a(P, sh, smem_u32(ring), off_dn + (has_dn ? ob : 0));
  {
    const int lane = threadIdx.x & 31;
    if (lane == 0) a.mine = rn_source(P.x, sizeof(TX), 0, P.dense & 1, D);
    if (lane == 1) a.mine = rn_source(P.o, sizeof(TO), xb, P.dense >> 1 & 1, D);
    if (GATE && lane == 2) a.mine = rn_source(P.g, sizeof(TO), off_g, P.dense >> 2 & 1, D);
    if (lane == 3) a.mine = rn_source(P.dv, sizeof(TX), off_dv, P.dense >> 3 & 1, D);
    if (lane == 4) a.mine = rn_source(P.dn, sizeof(TO), off_dn, P.dense >> 4 & 1, D);
  }
  float* params = reinterpret_cast<float*>(ring) + P.params;
  __syncthreads();
  a.start();
  rn_params(P, params);
  __syncthreads();
  unsigned long long seed = 0;
  if (DROP) seed = P.seed_ptr ? (unsigned long long)*P.seed_ptr : P.seed;
  const unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  const float inv = 1.f / D, keep = DROP ? P.keep_scale : 1.f;
  bool mine[K];
  u64 sw[K][H], sq[K][H];  // sums over this thread's rows: dw, Q
#pragma unroll
  for (int k = 0; k < K; ++k) {
    mine[k] = FULL || a.me * V + k * a.stride < D;
#pragma unroll
    for (int i = 0; i < H; ++i) sw[k][i] = sq[k][i] = 0ull;
  }
  const uint32_t at_x = a.sub * xb + a.me * (V * (uint32_t)sizeof(TX)), at_o = a.rows * xb + a.sub * ob + a.me * 16;
  const uint32_t to_dv = a.rows * off_dv, to_g = a.rows * (off_g - xb), to_dn = a.rows * (off_dn - xb);
  const uint32_t kx = a.stride * (uint32_t)sizeof(TX), ko = a.stride * (uint32_t)sizeof(TO), kp = a.stride * 4;
  const uint32_t pw = smem_u32(params) + a.me * V * 4, pws = pw + 4 * D;
  auto roots_of = [&](int row) {
    return row < a.total ? __ldg(reinterpret_cast<const float2*>(P.rstd + 2LL * row)) : make_float2(0.f, 0.f);
  };
  float2 ahead = roots_of(min(a.first, a.total) + a.sub);  // of the row to come
  for (int row0 = a.first; row0 < a.total; row0 += a.step) {
    a.wait();
    uint32_t px = a.base + a.slot * a.stage_bytes + at_x, po = a.base + a.slot * a.stage_bytes + at_o;
    int row = row0 + a.sub;
    for (int j = 0; j < a.batch && row - a.sub < a.total; ++j, row += a.per, px += a.per * xb, po += a.per * ob) {
      const bool here = !NARROW || row < a.total;
      const long long out = (long long)row * D + a.me * V;
      const float rb = ahead.x, r = ahead.y;
      ahead = roots_of(j + 1 < a.batch ? row + a.per : (int)min((long long)row0 + a.step, (long long)a.total) + a.sub);
      u64 v[K][H], s1 = 0ull, s2 = 0ull, s3 = 0ull;
      unsigned bits[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        bits[k] = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < H; ++i) v[k][i] = 0ull;
        if (mine[k] && here) {
          u64 f[H], t[H];
          rn_take<TO, V>(po + k * ko, t);
          rn_take<float, V>(pws + k * kp, f);
#pragma unroll
          for (int i = 0; i < H; ++i) t[i] = mul2(t[i], mul2(f[i], rn_all(rb)));
          if (GATE) {
            rn_take<TO, V>(po + to_g + k * ko, f);
#pragma unroll
            for (int i = 0; i < H; ++i) t[i] = mul2(t[i], rn_sigmoid(f[i]));
          }
          if (DROP) {
            bits[k] = rn_bits<V>(P, k0, k1, row, a.me * V + k * a.stride);
#pragma unroll
            for (int i = 0; i < H; ++i) t[i] = rn_mask(mul2(t[i], rn_all(keep)), bits[k], i);
          }
          rn_take<TX, V>(px + k * kx, f);
#pragma unroll
          for (int i = 0; i < H; ++i) v[k][i] = add2(f[i], t[i]);
          if (has_dn) {
            u64 q[H];
            rn_take<TO, V>(po + to_dn + k * ko, q);
            rn_take<float, V>(pw + k * kp, f);
#pragma unroll
            for (int i = 0; i < H; ++i) {
              q[i] = mul2(q[i], f[i]);
              s1 = fma2(q[i], v[k][i], s1);
              s2 = fma2(t[i], mul2(q[i], rn_all(r)), s2);
              s3 = fma2(t[i], v[k][i], s3);
            }
          }
          if (has_dv) {
            rn_take<TX, V>(px + to_dv + k * kx, f);
#pragma unroll
            for (int i = 0; i < H; ++i) s2 = fma2(t[i], f[i], s2);
          }
        }
      }
      float t[3] = {rn_hsum(s1), rn_hsum(s2), rn_hsum(s3)};
      a.sum(t);
      const float mean = t[0] * inv * r * r;                                 // of tw v, times r^2
      const float back = has_wb ? (t[1] - r * mean * t[2]) * inv * rb : 0.f;  // of t dv', times r_b
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (mine[k] && here) {
          u64 g[H], f[H], q[H], u[H], sg[H];  // g: gradient of the stream, then of less and less of the branch
#pragma unroll
          for (int i = 0; i < H; ++i) g[i] = 0ull;
          if (has_dn) {
            rn_take<TO, V>(po + to_dn + k * ko, q);
            rn_take<float, V>(pw + k * kp, f);
#pragma unroll
            for (int i = 0; i < H; ++i) {
              g[i] = mul2(rn_all(r), fma2(v[k][i], rn_all(-mean), mul2(f[i], q[i])));
              sw[k][i] = fma2(mul2(q[i], v[k][i]), rn_all(r), sw[k][i]);
            }
          }
          if (has_dv) {
            rn_take<TX, V>(px + to_dv + k * kx, f);
#pragma unroll
            for (int i = 0; i < H; ++i) g[i] = add2(g[i], f[i]);
          }
          rn_put<TX, V>(static_cast<TX*>(P.dx) + out + k * a.stride, g);
          if (DROP)
#pragma unroll
            for (int i = 0; i < H; ++i) g[i] = rn_mask(mul2(g[i], rn_all(keep)), bits[k], i);
          rn_take<TO, V>(po + k * ko, u);
          rn_take<float, V>(pws + k * kp, f);
          if (GATE) rn_take<TO, V>(po + to_g + k * ko, sg);
#pragma unroll
          for (int i = 0; i < H; ++i) {
            u64 n = mul2(u[i], rn_all(rb)), e = mul2(g[i], f[i]);
            if (DROP) n = rn_mask(n, bits[k], i);  // (a dropped element may hold anything)
            if (GATE) {
              const u64 s = rn_sigmoid(sg[i]), gs = DROP ? rn_mask(mul2(g[i], s), bits[k], i) : mul2(g[i], s);
              sq[k][i] = fma2(gs, n, sq[k][i]);
              const u64 es = mul2(gs, f[i]);
              sg[i] = mul2(mul2(es, n), rn_neg1_plus(s));
              if (DROP) sg[i] = rn_mask(sg[i], bits[k], i);
              e = es;
            } else {
              sq[k][i] = fma2(g[i], n, sq[k][i]);
            }
            if (has_wb) e = mul2(rn_all(rb), fma2(u[i], rn_all(-back), e));
            g[i] = e;
          }
          if (GATE) rn_put<TO, V>(static_cast<TO*>(P.dg) + out + k * a.stride, sg);
          rn_put<TO, V>(static_cast<TO*>(P.d_o) + out + k * a.stride, g);
        }
    }
    a.next(row0);
  }
  a.finish(P.err);
  // the CTA's sums: its threads of a channel in order (groups, then rows at once)
  __syncthreads();
  float* out = P.partial + (long long)blockIdx.x * 3 * D;
  const int groups = (int)(blockDim.x >> 5) / a.warps;
  for (int q = 0; q < groups * a.per; ++q) {
    if (a.group == q / a.per && a.sub == q % a.per)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = a.me * V + k * a.stride;
        if (mine[k])
#pragma unroll
          for (int i = 0; i < H; ++i) {
            u64* f0 = reinterpret_cast<u64*>(params + c) + i;
            u64* f1 = reinterpret_cast<u64*>(params + D + c) + i;
            *f0 = q ? add2(*f0, sw[k][i]) : sw[k][i];
            *f1 = q ? add2(*f1, sq[k][i]) : sq[k][i];
          }
      }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < D; i += blockDim.x) {
    out[i] = params[i];
    out[D + i] = params[D + i] * (P.scale ? P.scale[i] : 1.f);
    out[2 * D + i] = params[D + i] * (P.wb ? P.wb[i] : 1.f);
  }
}

// ---------------------------------------------------------------- backward, rows wherever they lie

// (The row's three sums, and what they are for, as in the kernel above.)
template <typename TX, typename TO, int K>
__global__ void __launch_bounds__(rn_plain_threads(K), K == 2 ? 2 : 1) rn_bwd_kernel(const __grid_constant__ RnParams P) {
  extern __shared__ __align__(16) float acc[];  // [groups][2][D] column sums of dw and Q (K = 2: at the end)
  __shared__ float part[2][3][RN_MAX_WARPS];
  int flip = 0;
  const int warps = P.warps, group = (threadIdx.x >> 5) / warps, groups = (blockDim.x >> 5) / warps;
  const int me = threadIdx.x - group * warps * 32, stride = warps * 128, c0 = me / 32 * 128 + me % 32;
  const unsigned long long seed = P.seed_ptr ? (unsigned long long)*P.seed_ptr : P.seed;
  const unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  const float inv = 1.f / P.D;
  float* sums = acc + group * 2 * P.D;
  float mine[2][K][4] = {};  // (K = 2)
  if (K > 2)
#pragma unroll
    for (int k = 0; k < K; ++k)
      for (int i = 0; i < rn_there(c0 + k * stride, P.D); ++i)
        for (int q = 0; q < 2; ++q) sums[q * P.D + c0 + k * stride + 32 * i] = 0.f;
  auto add = [&](int q, int k, int c, int n, const float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (K == 2) mine[q][k][i] += f[i];
      else if (i < n) sums[q * P.D + c + 32 * i] += f[i];
    }
  };
  for (long long row = (long long)blockIdx.x * groups + group; row < P.rows; row += (long long)gridDim.x * groups) {
    const TX* px = rn_row<TX>(P.x, row, P.T);
    const TO* po = rn_row<TO>(P.o, row, P.T);
    const TO* pg = P.g.p ? rn_row<TO>(P.g, row, P.T) : nullptr;
    const TX* pdv = P.dv.p ? rn_row<TX>(P.dv, row, P.T) : nullptr;
    const TO* pdn = P.dn.p ? rn_row<TO>(P.dn, row, P.T) : nullptr;
    RnFour<TO> o[K], g[K], dn[K];
    RnFour<TX> x[K], dv[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = c0 + k * stride, n4 = rn_there(c, P.D);
      o[k].load(po + c, n4);
      x[k].load(px + c, n4);
      if (pg) g[k].load(pg + c, n4);
      dv[k].load(pdv + c, pdv ? n4 : 0);
      dn[k].load(pdn + c, pdn ? n4 : 0);
    }
    const float rb = P.rstd[2 * row], r = P.rstd[2 * row + 1];
    // the stream again, and the row's sums (as above)
    float v[K][4], sum[3] = {0.f, 0.f, 0.f};
    unsigned kept[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = c0 + k * stride, n4 = rn_there(c, P.D);
      kept[k] = P.dropout ? rn_kept(P, k0, k1, row, c) : 15u;
      float f[4], t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = o[k].get(i);
      if (P.wb) {
        rn_param(P.wb, c, n4, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] *= rb * f[i];
      }
      if (pg)
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] *= sigmoidf_(g[k].get(i));
      if (P.scale) {
        rn_param(P.scale, c, n4, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] *= f[i];
      }
      if (P.dropout)
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = kept[k] >> i & 1 ? P.keep_scale * t[i] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = 0.f;
      if (pdn) rn_param(P.w, c, n4, f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[k][i] = x[k].get(i) + t[i];
        const float q = f[i] * dn[k].get(i);
        sum[0] = fmaf(q, v[k][i], sum[0]);
        sum[1] = fmaf(t[i], fmaf(r, q, dv[k].get(i)), sum[1]);
        sum[2] = fmaf(t[i], v[k][i], sum[2]);
      }
    }
    if (pdn || P.wb) rn_sum(sum, part[flip ^= 1], group, warps);
    const float mean = sum[0] * inv * r * r, back = P.wb ? (sum[1] - r * mean * sum[2]) * inv * rb : 0.f;
    TX* pdx = static_cast<TX*>(P.dx) + row * P.D;
    TO* pdg = static_cast<TO*>(P.dg) + row * P.D;
    TO* pdo = static_cast<TO*>(P.d_o) + row * P.D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = c0 + k * stride, n4 = rn_there(c, P.D);
      float d[4], f[4], t[4], wb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = dv[k].get(i);
      if (pdn) {
        rn_param(P.w, c, n4, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d[i] = fmaf(r, fmaf(-v[k][i], mean, f[i] * dn[k].get(i)), d[i]);
          t[i] = dn[k].get(i) * v[k][i] * r;
        }
        add(0, k, c, n4, t);
      }
      rn_store(pdx + c, d, n4);
      if (P.wb) rn_param(P.wb, c, n4, wb);
      if (P.scale) rn_param(P.scale, c, n4, f);
      float s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool on = kept[k] >> i & 1;
        const float n = o[k].get(i) * rb;
        s[i] = pg ? sigmoidf_(g[k].get(i)) : 1.f;
        const float gs = on ? (P.dropout ? P.keep_scale * d[i] : d[i]) * s[i] : 0.f;
        t[i] = on ? gs * n : 0.f;
        d[i] = on ? gs * ((P.scale ? f[i] : 1.f) * (P.wb ? wb[i] : 1.f)) : 0.f;
        s[i] = on ? d[i] * n * (1.f - s[i]) : 0.f;
        if (P.wb) d[i] = rb * fmaf(-o[k].get(i), back, d[i]);
      }
      add(1, k, c, n4, t);
      if (pg) rn_store(pdg + c, s, n4);
      rn_store(pdo + c, d, n4);
    }
  }
  if (K == 2)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < rn_there(c0 + k * stride, P.D))
#pragma unroll
          for (int q = 0; q < 2; ++q) sums[q * P.D + c0 + k * stride + 32 * i] = mine[q][k][i];
  __syncthreads();
  float* out = P.partial + (long long)blockIdx.x * 3 * P.D;
  for (int i = threadIdx.x; i < P.D; i += blockDim.x) {  // the CTA's sums, its groups in order
    float t = 0.f, q = 0.f;
    for (int w = 0; w < groups; ++w) t += acc[w * 2 * P.D + i], q += acc[(w * 2 + 1) * P.D + i];
    out[i] = t;
    out[P.D + i] = q * (P.scale ? P.scale[i] : 1.f);
    out[2 * P.D + i] = q * (P.wb ? P.wb[i] : 1.f);
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
