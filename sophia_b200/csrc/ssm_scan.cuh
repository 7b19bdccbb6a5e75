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
// Layout.  Time runs in order: a channel's N states are spread over L lanes with S
// states each (L S >= N), its recurrence stays in registers, and 32 / L channels
// share a warp.  The decay's exponential (16 a clock and SM) is evaluated once per
// token, channel and state.  Four warps run the recurrences of a tile of tokens while
// four others do what depends on the token and channel alone: they fetch the tile
// after the next (cp.async), turn the next one into d, d x and fp32 rows of B and C
// (softplus, gates), and finish the one before (sum of the lanes' parts, skip, gate,
// store).  The two sides exchange double buffers in shared memory, one barrier per tile.
//
// Backward.  Tiles from last to first, in segments of SCAN_SEG tokens: a segment's
// states are rebuilt from the checkpoint that the forward saved at its start and kept in
// registers with their decays, then its tokens run backwards.  dB and dC are sums
// over channels: the lanes of one warp that hold the same states of different channels
// exchange halves of their values (each lane orders its states by its channel, n = n0 +
// (i xor m), so that what a lane keeps sits in the same registers everywhere), the
// warps' sums meet in shared memory and the CTAs' in a buffer that a last kernel sums in
// block order.  No atomics: every sum has a fixed order.
//
// Few rows: the tokens are cut into spans with CTAs of their own.  As h is linear in the
// state in front, a span's effect on it is h -> P h + c, P = e^(A sum d) and c the state that
// the span makes of zeros; a first kernel finds P and c of every span (the recurrence
// alone: no C, no output), and a CTA of the scan itself composes those in front of its own.
// Backward the same with g, from behind.
//
// What bounds it: latency, neither HBM nor a pipe.  For 32 states' tokens (N = 16) the forward issues 10
// instructions and holds the exponentials' pipe for 2.5 cycles of 4.2; the backward 32 and 4.3 of 11, half of
// the instructions on the token side.  Counters, bf16, 4 x 4096 tokens x 2048 channels, N = 16 (256 CTAs: 108 SMs with
// two, 40 with one): forward 53 % of issue slots, 53 % of that pipe, 71 % of shared memory, 3.4 warps per
// scheduler of which 0.8 can issue, none in 47 % of cycles; backward 62 %, 30 %, 60 %, 3.3 warps, 1.1, 38 %.  Of the
// 6.4 and 5.4 cycles between a warp's instructions 1.9 and 1.3 are fixed latency, 1.3 and 0.5 shared memory and
// special functions, 0.5 and 0.7 the barrier of the tile.
// Measured there: forward 302 us (0.9 TB/s; 285 without checkpoints), backward 796 + 31 us for dB and dC; 8192 packed tokens in
// 9 spans 150 + 114 (carries) forward, 392 + 114 backward; a prompt of 16384 tokens 262 + 193.
#pragma once

#include <cfloat>

#include "ssm_common.cuh"

namespace kda {

constexpr int SCAN_MAIN = 128;                // threads with recurrences
constexpr int SCAN_WARPS = SCAN_MAIN / 32;
constexpr int SCAN_TOKENS = 128;              // threads of the token side
constexpr int SCAN_THREADS = SCAN_MAIN + SCAN_TOKENS;
constexpr int SCAN_SEG = 8;      // tokens between checkpoints
constexpr int SCAN_TT_BWD = 8;   // tokens per tile of the backward
constexpr int SCAN_STAGES = 4;   // raw tiles in shared memory

__host__ __device__ constexpr int ilog2(int v) { return v <= 1 ? 0 : 1 + ilog2(v / 2); }

// Geometry of a variant: L lanes per channel, S states per lane, tiles of TT tokens.
template <typename T, int L_, int S_, int TT_>
struct ScanGeo {
  static constexpr int L = L_, S = S_, TT = TT_, TOKENS = SCAN_TOKENS;
  static constexpr int NP = L * S;               // states with padding
  static constexpr int CH = 32 / L;              // channels per warp
  static constexpr int CPB = SCAN_WARPS * CH;    // channels per CTA
  static constexpr int RAW = TT * CPB;           // elements of a staged tensor
  static constexpr int PAIRS = CPB / 2;          // channel pairs: a thread's share of a token pass
  static constexpr int TSTEP = TOKENS / PAIRS < TT ? TOKENS / PAIRS : TT;  // tokens per pass of the side
  static constexpr bool SPARE = TOKENS / PAIRS > TT;  // threads without a token
  static constexpr int V = 16 / (int)sizeof(T), NV = CPB / V;  // 16-byte pieces of a row
  // partial sums over the lanes, [TT][L][CPB and a pad]: neither the lanes' stores nor the reads of channel
  // pairs share a bank
  static constexpr int YS = CPB + CH, YT = L * YS;
  // the backward's S versions of B and C, [TT][S and a pad][NP], likewise
  static constexpr int BS = (S + 1) * NP;
};
// Tiles of the carries' kernel; the forward's are scan_cut's choice.
template <typename T, int L, int S>
using ScanCarryGeo = ScanGeo<T, L, S, (sizeof(T) == 2 && L > 2) ? 32 : 16>;
template <typename T, int L, int S>
using ScanBwdGeo = ScanGeo<T, L, S, SCAN_TT_BWD>;

struct ScanParams {
  RowView x, dt, z, dy;            // [B, T, E]; z.p null = no gate
  const void *Bm, *Cm;             // [B, T, G, N], rows of N contiguous
  long long b_sb, b_st, b_sg, c_sb, c_st, c_sg;
  const float *A, *D, *dt_bias;    // [E][N], [E] or null, [E] or null
  const float* h0;                 // [nseq][E][N] or null
  SeqMap seq;
  int B, T, E, N, G;
  int blocks;                      // channel blocks per group
  int spans, span;                 // of `span` tokens (a multiple of 32)
  int tile;                        // tokens of a forward tile
  float2* carry;                   // [B][spans][E][N]: c and P (negative: nothing passes) of the spans; null = one span
  bool softplus, vec, vec_bc;      // vec: x, dt, z, dy and the outputs allow 16-byte pieces; vec_bc: B and C
  void* y;                         // [B, T, E] contiguous
  float* ht;                       // [nseq][E][N] or null
  float* ckpt;                     // [B][segments][E][N]: states in front of each segment; null = not kept
  // backward
  const float* dht;
  void *dx, *ddt, *dz;
  float* dh0;
  float* bc_part;                  // [B][tiles][G][blocks][TT][2][N]
  float* e_part;                   // [B][spans][E][N + 2]: dA, dD, d dt_bias
};

struct ScanBlock {
  int g, blk, c0, nc, b;  // group, block in it, first channel, channels, row
  int k;                  // span
  int tile0, tiles;       // its tiles
};
template <int CPB, int TT>
__device__ __forceinline__ ScanBlock scan_block(const ScanParams& P, int span) {
  ScanBlock s;
  const int eg = P.E / P.G;
  s.g = blockIdx.x / P.blocks;
  s.blk = blockIdx.x - s.g * P.blocks;
  s.c0 = s.g * eg + s.blk * CPB;
  s.nc = min(CPB, eg - s.blk * CPB);
  s.b = blockIdx.y;
  s.k = span;
  s.tile0 = span * (P.span / TT);
  s.tiles = (min(P.span, P.T - span * P.span) + TT - 1) / TT;
  return s;
}

// The decays 2^(d a2).  ex2.approx is low by 0.5e-8 to 2.9e-8 on average where decays are close
// to 1 (measured: 0.5e-8 for exponents of -3e-4 to -3e-3, 2.4e-8 for -0.005 to -0.08, 1.8e-8 for
// -0.08 to -0.3), which adds up over the tokens that a state remembers.  An exponent
// raised by 1e-8 / ln 2 takes the middle of that off, at no cost (an fma for a product); 2^0
// stays 1.
constexpr float SCAN_EXP_SHIFT = 1.44e-8f;
template <int S>
__device__ __forceinline__ Lane<S> lane_decay(const Lane<S>& a2, float d) {
  return fma(a2, Lane<S>::all(d), Lane<S>::all(SCAN_EXP_SHIFT)).exp2();
}
// A decay rate in powers of two, for the backward.  A state that forgets at once (a rate of -inf) has the lowest finite
// one: 2^(d a2) is 0 for every d above 1e-36 all the same, and 1 for the d = 0 of the places past a row's end,
// where 0 x inf would make NaN of the gradients that the backward carries on from there (nothing is carried from
// there forward).
__device__ __forceinline__ float scan_rate(float a) {
  const float v = a * LOG2E;
  return v == -INFINITY ? -FLT_MAX : v;
}
// sum += v with the rounding errors carried along (a compensated sum: its error does not
// grow with the number of tokens).
__device__ __forceinline__ void sum_add(float& sum, float& err, float v) {
  const float y = __fadd_rn(v, -err), t = __fadd_rn(sum, y);
  err = __fadd_rn(__fadd_rn(t, -sum), -y);
  sum = t;
}

// Zero in the states that do not exist (PAD: N < L S), whatever arithmetic made of them.
template <bool PAD, int S>
__device__ __forceinline__ Lane<S> lane_keep(Lane<S> v, unsigned ok) {
  if (PAD) {
#pragma unroll
    for (int i = 0; i < S; ++i) v.set(i, ok >> i & 1 ? v.get(i) : 0.f);
  }
  return v;
}

__device__ __forceinline__ void cp_async8(void* smem, const void* gmem, bool pred) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(smem_u32(smem)), "l"(gmem), "r"(pred ? 8 : 0)
               : "memory");
}

// The token side's fetches.  Every thread keeps where its pieces of a tile come from
// (the aligned case: 16-byte pieces by cp.async, zeros past T and, whole pieces, past the
// block's channels); else elements are copied one by one.  Rows of B and C likewise.
template <typename T, typename G, int TENSORS>
struct ScanFetch {
  static constexpr int PIECES = G::TT * G::NV, SLOTS = (TENSORS * PIECES + G::TOKENS - 1) / G::TOKENS;
  static constexpr int BC_SLOTS = (2 * G::TT * (G::NP < G::V ? 1 : G::NP / G::V) + G::TOKENS - 1) / G::TOKENS;
  static constexpr int SL = SLOTS > 0 ? SLOTS : 1;
  const T* src[SL];      // the piece in the tile to come
  const T* safe[SL];     // an address to name where nothing is read
  long long step[SL];    // elements to the next tile
  int dst[SL], row[SL];  // token in the tile; far past it: zeros
  const T* bc_src[BC_SLOTS];
  int bc_dst[BC_SLOTS], bc_row[BC_SLOTS];
  long long bc_step[BC_SLOTS];

  // `tile` is fetched first, then its neighbour in direction `dir`, and so on.
  __device__ __forceinline__ void init(const ScanParams& P, const ScanBlock& s, const RowView (&r)[TENSORS], int tid,
                                       int bc_at, int npad, int tile, int dir) {
    const long long t0 = (long long)tile * G::TT;
    if (P.vec) {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k) {
        const int i = k * G::TOKENS + tid, w = i / PIECES, j = i - w * PIECES;
        row[k] = j / (G::NV > 0 ? G::NV : 1);
        const int c = (j - row[k] * G::NV) * G::V;
        src[k] = safe[k] = nullptr;
        step[k] = 0;
        dst[k] = w * G::RAW + row[k] * G::CPB + c;
#pragma unroll
        for (int q = 0; q < TENSORS; ++q)
          if (w == q && r[q].p) {
            safe[k] = static_cast<const T*>(r[q].p);
            src[k] = safe[k] + s.b * r[q].sb + (t0 + row[k]) * r[q].st + s.c0 + c;
            step[k] = dir * G::TT * r[q].st;
          }
        if (c >= s.nc) row[k] = 1 << 30;  // past the channels: zeros
      }
    }
    if (P.vec_bc) {
      const int nv = P.N < G::V ? 1 : P.N / G::V, per = G::TT * nv;
#pragma unroll
      for (int k = 0; k < BC_SLOTS; ++k) {
        const int i = k * G::TOKENS + tid, w = i / per, j = i - w * per;
        bc_row[k] = j / nv;
        const int n = (j - bc_row[k] * nv) * G::V;
        bc_src[k] = nullptr;
        if (w == 0) bc_src[k] = static_cast<const T*>(P.Bm) + s.b * P.b_sb + s.g * P.b_sg + (t0 + bc_row[k]) * P.b_st + n;
        if (w == 1) bc_src[k] = static_cast<const T*>(P.Cm) + s.b * P.c_sb + s.g * P.c_sg + (t0 + bc_row[k]) * P.c_st + n;
        bc_step[k] = dir * G::TT * (w ? P.c_st : P.b_st);
        bc_dst[k] = bc_at + w * G::TT * npad + bc_row[k] * P.N + n;
      }
    }
  }
  __device__ __forceinline__ void fetch(const ScanParams& P, const ScanBlock& s, const RowView (&r)[TENSORS], T* stage, int t0,
                                        int tid) {
    if (P.vec) {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k)
        if (safe[k]) {
          const bool in = row[k] < P.T - t0;
          cp_async16(stage + dst[k], in ? src[k] : safe[k], in);
          src[k] += step[k];
        }
    } else {
#pragma unroll
      for (int q = 0; q < TENSORS; ++q)
        if (r[q].p)
          for (int i = tid; i < G::TT * G::CPB; i += G::TOKENS) {
            const int t = i / G::CPB, c = i - t * G::CPB;
            stage[q * G::RAW + i] =
                t0 + t < P.T && c < s.nc ? row_ptr<T>(r[q], s.b, t0 + t)[s.c0 + c] : io_from_f<T>(0.f);
          }
    }
    if (P.vec_bc) {
#pragma unroll
      for (int k = 0; k < BC_SLOTS; ++k)
        if (bc_src[k]) {
          const bool in = bc_row[k] < P.T - t0;
          const T* src_bc = in ? bc_src[k] : static_cast<const T*>(P.Bm);
          if (P.N < G::V) cp_async8(stage + bc_dst[k], src_bc, in);
          else cp_async16(stage + bc_dst[k], src_bc, in);
          bc_src[k] += bc_step[k];
        }
    }
    cp_async_commit();
  }
};
// vec_bc: rows of B and C are whole 16-byte pieces, or the 8 bytes of four 16-bit states.
// vec: a block's channels are whole 16-byte pieces, or end with the tensor's row
// (E a multiple of the piece), so a piece never mixes two blocks' channels.

// B and C of a tile as fp32 [TT][VERS][NP], version v holding state n0 + (i ^ v) at n0 + i of a
// lane's S states (zeros past T and past N); from the staged rows or from global memory.
// Reads (load) and writes (store) apart, as the compiler must assume that they alias.
template <typename T, typename G, int VERS, bool PAD>
struct ScanBC {
  static constexpr int ITEMS = 2 * G::TT * G::L, SLOTS = (ITEMS + G::TOKENS - 1) / G::TOKENS;
  float v[SLOTS][G::S];
  __device__ __forceinline__ void load(const T* raw, int npad, const ScanParams& P, const ScanBlock& s, int t0, int tid) {
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      const int i = k * G::TOKENS + tid;
      if (ITEMS % G::TOKENS != 0 && i >= ITEMS) break;
      const bool is_c = i >= G::TT * G::L;
      const int j = is_c ? i - G::TT * G::L : i, t = j / G::L, n0 = (j - t * G::L) * G::S;
      if (P.vec_bc && !PAD) {
        io_load<T, G::S>(raw + (is_c ? G::TT * npad : 0) + t * P.N + n0, v[k]);
        continue;
      }
#pragma unroll
      for (int q = 0; q < G::S; ++q) {
        v[k][q] = 0.f;
        if (n0 + q < P.N) {
          if (P.vec_bc) {
            v[k][q] = io_to_f(raw[(is_c ? G::TT * npad : 0) + t * P.N + n0 + q]);
          } else if (t0 + t < P.T) {
            const T* p = is_c ? static_cast<const T*>(P.Cm) + s.b * P.c_sb + s.g * P.c_sg + (t0 + t) * P.c_st
                              : static_cast<const T*>(P.Bm) + s.b * P.b_sb + s.g * P.b_sg + (t0 + t) * P.b_st;
            v[k][q] = io_to_f(p[n0 + q]);
          }
        }
      }
    }
  }
  __device__ __forceinline__ void store(float* Bs, float* Cs, int tid) const {
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      const int i = k * G::TOKENS + tid;
      if (ITEMS % G::TOKENS != 0 && i >= ITEMS) break;
      const bool is_c = i >= G::TT * G::L;
      const int j = is_c ? i - G::TT * G::L : i, t = j / G::L, n0 = (j - t * G::L) * G::S;
      float* dst = is_c ? Cs : Bs;
#pragma unroll
      for (int w = 0; w < VERS; ++w) {
        IoVec<float, G::S> o;
#pragma unroll
        for (int q = 0; q < G::S; ++q) o.v[q] = v[k][q ^ w];
        *reinterpret_cast<IoVec<float, G::S>*>(dst + t * (VERS == 1 ? G::NP : G::BS) + w * G::NP + n0) = o;
      }
    }
  }
};

// Pair of neighbouring channels of a staged row.
template <typename T>
__device__ __forceinline__ float2 scan_pair(const T* p) {
  float f[2];
  io_load<T, 2>(p, f);
  return make_float2(f[0], f[1]);
}
// Stores a pair of channels of a [B, T, E] output at element `at`: how is 2 for both at once, 1 one by one,
// bit 2 without the first and bit 3 without the second.
template <typename T>
__device__ __forceinline__ void scan_put_pair(void* out, long long at, int how, float2 v) {
  T* p = static_cast<T*>(out) + at;
  if (how == 2) {
    const float f[2] = {v.x, v.y};
    io_store<T, 2>(p, f);
  } else {
    if (!(how & 4)) p[0] = io_from_f<T>(v.x);
    if (!(how & 8)) p[1] = io_from_f<T>(v.y);
  }
}
__device__ __forceinline__ int scan_how(const ScanParams& P, const ScanBlock& s, int c) {
  return P.vec && c + 1 < s.nc ? 2 : 1 | (c < s.nc ? 0 : 4) | (c + 1 < s.nc ? 0 : 8);
}
// Sums of a channel pair's L partial sums.
template <typename G>
__device__ __forceinline__ float2 scan_join(const float* p) {
  u64 acc = *reinterpret_cast<const u64*>(p);
#pragma unroll
  for (int l = 1; l < G::L; ++l) acc = add2(acc, *reinterpret_cast<const u64*>(p + l * G::YS));
  return upk2(acc);
}

// d of a token, 0 past the row's end.
__device__ __forceinline__ float scan_d(const ScanParams& P, float raw, bool inside) {
  const float d = P.softplus ? softplusf_(raw) : raw;
  return inside ? d : 0.f;
}

// First and last tokens of sequences: thread tid < TT looks after token tid of the tiles, a
// tile ahead of the place in shared memory ([TT] first, [TT] last) that it goes to.
template <int TT>
struct ScanFlags {
  int f, l;
  __device__ __forceinline__ void read(const ScanParams& P, int b, int t0, int tid) {
    if (tid >= 32) return;  // (TT <= 32: the first warp's)
    const int t = t0 + tid;
    const bool in = tid < TT && t >= 0 && t < P.T;
    f = in ? seq_start_at(P.seq, b, t) : -1;
    l = in ? seq_end_at(P.seq, b, t) : -1;
  }
  __device__ __forceinline__ void write(int* flags, int tid) const {
    if (tid < TT) {
      flags[tid] = f;
      flags[TT + tid] = l;
    }
  }
};
__device__ __forceinline__ bool scan_seg_flag(const int* first, const int* last) {
  bool any = false;
#pragma unroll
  for (int k = 0; k < SCAN_SEG; k += 4) {
    const int4 f = *reinterpret_cast<const int4*>(first + k), l = *reinterpret_cast<const int4*>(last + k);
    any |= (f.x & f.y & f.z & f.w & l.x & l.y & l.z & l.w) >= 0;  // -1 everywhere: no flag
  }
  return any;
}

template <typename T, typename G>
__host__ __device__ inline int scan_stage_elems(int N, int tensors) {
  return tensors * G::RAW + 2 * G::TT * ((N + 7) / 8 * 8);
}
template <typename T, typename G>
__host__ __device__ inline int scan_fwd_smem(int N) {
  return SCAN_STAGES * scan_stage_elems<T, G>(N, 3) * (int)sizeof(T) +
         2 * (G::TT * G::CPB * 8 + 2 * G::TT * G::NP * 4 + G::TT * G::YT * 4 + 2 * G::TT * 4);
}
template <typename T, typename G>
__host__ __device__ inline int scan_bwd_smem(int N) {
  return SCAN_STAGES * scan_stage_elems<T, G>(N, 4) * (int)sizeof(T) +
         3 * G::TT * G::CPB * 16 + 2 * (2 * G::TT * G::BS * 4 + 3 * G::TT * G::YT * 4 +
                                        SCAN_WARPS * G::TT * 2 * G::NP * 4 + 2 * G::TT * 4);
}

template <typename T, typename G>
__host__ __device__ inline int scan_carry_smem(int N, int tensors) {
  return SCAN_STAGES * scan_stage_elems<T, G>(N, tensors) * (int)sizeof(T) +
         2 * (G::TT * G::CPB * 8 + 2 * G::TT * G::NP * 4 + 2 * G::TT * 4);
}

// A channel pair's values of a per-channel parameter (zeros without it or past the block).
__device__ __forceinline__ float2 scan_param(const float* p, const ScanBlock& s, int c) {
  return make_float2(p && c < s.nc ? p[s.c0 + c] : 0.f, p && c + 1 < s.nc ? p[s.c0 + c + 1] : 0.f);
}

// A lane's states of sequence q, register i being state i ^ m of the lane's (zeros where `ok` has no
// bit, and without the tensor).
template <int S>
__device__ __forceinline__ Lane<S> scan_state(const float* states, int q, long long per, long long chan, unsigned ok, int m) {
  float f[S];
#pragma unroll
  for (int i = 0; i < S; ++i) f[i] = 0.f;
  if (states && ok) {
    const float* p = states + q * per + chan;
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (ok >> i & 1) f[i] = p[i ^ m];
  }
  return Lane<S>::of(f);
}

// What the spans in front of span k (REV: behind it) hand over: state n of a lane's register i
// at chan + (i ^ m).  A product with a zero is left out, so that P may be infinite.
template <int S, bool REV>
__device__ __forceinline__ Lane<S> scan_enter(const ScanParams& P, const ScanBlock& s, long long chan, unsigned ok, int m) {
  constexpr int U = 4;  // loads of four spans at once
  const long long per = (long long)P.E * P.N, step = REV ? -per : per;
  const int n = REV ? P.spans - 1 - s.k : s.k;
  const float2* p = P.carry + ((long long)s.b * P.spans + (REV ? P.spans - 1 : 0)) * per + chan;
  float v[S];
#pragma unroll
  for (int i = 0; i < S; ++i) v[i] = 0.f;
  for (int j = 0; j < n; j += U, p += U * step) {
    float2 c[U][S];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < S; ++i)
        c[u][i] = j + u < n && (ok >> i & 1) ? __ldg(p + u * step + (i ^ m)) : make_float2(0.f, 1.f);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < S; ++i) v[i] = c[u][i].y < 0.f || v[i] == 0.f ? c[u][i].x : fmaf(c[u][i].y, v[i], c[u][i].x);
  }
  return Lane<S>::of(v);
}

// P and c of the spans that have one behind them (REV: in front, for the backward's g, where
// u = dy silu(z) and C stand for d x and B).  The same layout as the scan's, without its outputs.
template <typename T, int L, int S, bool PAD, bool REV>
__global__ void __launch_bounds__(SCAN_THREADS, 3) ssm_scan_carry_kernel(ScanParams P) {
  using G = ScanCarryGeo<T, L, S>;
  constexpr int TT = G::TT, CPB = G::CPB, TENSORS = REV ? 3 : 2;
  extern __shared__ __align__(16) char scan_sm[];
  const int N = P.N, npad = (N + 7) / 8 * 8, stage = scan_stage_elems<T, G>(N, TENSORS);
  T* raw = reinterpret_cast<T*>(scan_sm);                             // [STAGES]: dt, x or (dy, z), B rows, C rows
  float2* DU = reinterpret_cast<float2*>(raw + SCAN_STAGES * stage);  // double buffers: [TT][CPB]: d, u
  float* Bs = reinterpret_cast<float*>(DU + 2 * TT * CPB);            // [TT][NP]
  float* Cs = Bs + 2 * TT * G::NP;
  int* flags = reinterpret_cast<int*>(Cs + 2 * TT * G::NP);           // first [TT], last [TT]
  const ScanBlock s = scan_block<CPB, TT>(P, blockIdx.z + (REV ? 1 : 0));
  const int tiles = s.tiles, dir = REV ? -1 : 1, tile0 = REV ? s.tile0 + tiles - 1 : s.tile0;  // step i takes tile0 + i dir

  if (threadIdx.x >= SCAN_MAIN) {  // tokens
    const int tid = threadIdx.x - SCAN_MAIN;
    const int pc = (tid % G::PAIRS) * 2, pt = tid / G::PAIRS;
    const float2 bias = scan_param(P.dt_bias, s, pc);
    RowView views[TENSORS];
    views[0] = P.dt;
    views[1] = REV ? P.dy : P.x;
    if (REV) views[TENSORS - 1] = P.z;
    ScanFetch<T, G, TENSORS> f;
    f.init(P, s, views, tid, TENSORS * G::RAW, npad, tile0, dir);
    ScanFlags<TT> marks;
    marks.read(P, s.b, tile0 * TT, tid);
    constexpr int IT = TT / G::TSTEP;
    const bool spare = G::SPARE && pt >= TT;
    auto prepare = [&](int i) {
      const int t0 = (tile0 + i * dir) * TT, q = i & 1;
      const T* rx = raw + (i % SCAN_STAGES) * stage;
      ScanBC<T, G, 1, PAD> bc;
      float4 du[IT];
      if (!spare) {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          const int t = pt + k * G::TSTEP;
          const T* p = rx + t * CPB + pc;
          const float2 dt = scan_pair(p);
          float2 u = scan_pair(p + G::RAW);
          const bool in = t0 + t < P.T;
          const float d0 = scan_d(P, dt.x + bias.x, in), d1 = scan_d(P, dt.y + bias.y, in);
          if (!REV) {
            u.x *= d0;
            u.y *= d1;
          } else if (P.z.p) {
            const float2 z = scan_pair(p + 2 * G::RAW);
            u.x *= z.x * sigmoidf_(z.x);
            u.y *= z.y * sigmoidf_(z.y);
          }
          du[k] = make_float4(d0, u.x, d1, u.y);
        }
      }
      bc.load(rx + TENSORS * G::RAW, npad, P, s, t0, tid);
      if (!spare) {
#pragma unroll
        for (int k = 0; k < IT; ++k)
          *reinterpret_cast<float4*>(DU + (q * TT + pt + k * G::TSTEP) * CPB + pc) = du[k];
      }
      bc.store(Bs + q * TT * G::NP, Cs + q * TT * G::NP, tid);
      marks.write(flags + q * 2 * TT, tid);
      marks.read(P, s.b, t0 + dir * TT, tid);
    };
    f.fetch(P, s, views, raw, tile0 * TT, tid);
    if (tiles > 1) f.fetch(P, s, views, raw + stage, (tile0 + dir) * TT, tid);
    cp_async_wait<0>();
    asm volatile("bar.sync 1, %0;" ::"n"(G::TOKENS) : "memory");  // the first tiles have arrived, for the whole side
    prepare(0);
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      if (i + 2 < tiles) f.fetch(P, s, views, raw + ((i + 2) % SCAN_STAGES) * stage, (tile0 + (i + 2) * dir) * TT, tid);
      if (i + 1 < tiles) prepare(i + 1);
      cp_async_wait<0>();
      __syncthreads();
    }
    return;
  }

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane / G::CH, c = warp * G::CH + lane % G::CH, n0 = l * S;
  const unsigned ok = N - n0 >= S ? (1u << S) - 1u : N > n0 ? (1u << (N - n0)) - 1u : 0u;  // states that exist
  const bool live = c < s.nc;
  Lane<S> a2 = Lane<S>::all(0.f), h = a2;
  const long long chan = (long long)(s.c0 + (live ? c : 0)) * N + n0;
#pragma unroll
  for (int i = 0; i < S; ++i)
    if (live && (ok >> i & 1)) a2.set(i, REV ? scan_rate(P.A[chan + i]) : P.A[chan + i] * LOG2E);
  float dsum = 0.f, dsum_err = 0.f;
  bool cut = false;  // a sequence starts in the span: nothing passes it
  __syncthreads();
  for (int step = 0; step < tiles; ++step) {
    const int t0 = (tile0 + step * dir) * TT, q = step & 1;
    const float2* du_ = DU + q * TT * CPB + c;
    const float* v_ = (REV ? Cs : Bs) + q * TT * G::NP + n0;
    const int* first = flags + q * 2 * TT;
    const int* last = first + TT;
    float d;
    auto token = [&](float2 u, const Lane<S>& v) {
      const Lane<S> a = lane_decay(a2, u.x);
      d += u.x;
      if (!REV) h = lane_keep<PAD>(fma(a, h, v * Lane<S>::all(u.y)), ok);
      else h = a * lane_keep<PAD>(fma(v, Lane<S>::all(u.y), h), ok);
    };
    auto segment = [&](int t1) {
      float2 du[SCAN_SEG];
      Lane<S> v[SCAN_SEG];
#pragma unroll
      for (int k = 0; k < SCAN_SEG; ++k) {
        du[k] = du_[(t1 + k) * CPB];
        v[k] = Lane<S>::load(v_ + (t1 + k) * G::NP);
      }
#pragma unroll
      for (int o = 0; o < SCAN_SEG; ++o) token(du[REV ? SCAN_SEG - 1 - o : o], v[REV ? SCAN_SEG - 1 - o : o]);
    };
    auto flagged = [&](int t1) {  // sequences start or end among the tokens
      const long long per = (long long)P.E * N;
#pragma unroll 1
      for (int o = 0; o < SCAN_SEG; ++o) {
        const int t = t1 + (REV ? SCAN_SEG - 1 - o : o);
        const bool starts = first[t] >= 0;
        cut |= starts;
        if (!REV && starts) h = scan_state<S>(P.h0, first[t], per, chan, live ? ok : 0u, 0);
        if (REV && last[t] >= 0) h = h + scan_state<S>(P.dht, last[t], per, chan, live ? ok : 0u, 0);
        token(du_[t * CPB], Lane<S>::load(v_ + t * G::NP));
        if (REV && starts) h = Lane<S>::all(0.f);
      }
    };
    const int segs = (min(TT, P.T - t0) + SCAN_SEG - 1) / SCAN_SEG;
#pragma unroll 1
    for (int j = 0; j < segs; ++j) {
      const int t1 = (REV ? segs - 1 - j : j) * SCAN_SEG;
      d = 0.f;
      if (scan_seg_flag(first + t1, last + t1)) flagged(t1);
      else segment(t1);
      sum_add(dsum, dsum_err, d);
    }
    __syncthreads();
  }
  const Lane<S> pass = (a2 * Lane<S>::all(dsum)).exp2();
  float2* out = P.carry + ((long long)s.b * P.spans + s.k) * P.E * N + chan;
#pragma unroll
  for (int i = 0; i < S; ++i)
    if (live && (ok >> i & 1)) out[i] = make_float2(h.get(i), cut ? -1.f : pass.get(i));
}

template <typename T, int L, int S, int TT, bool PAD>
__global__ void __launch_bounds__(SCAN_THREADS, 2) ssm_scan_fwd_kernel(ScanParams P) {
  using G = ScanGeo<T, L, S, TT>;
  constexpr int CPB = G::CPB;
  extern __shared__ __align__(16) char scan_sm[];
  const int N = P.N, npad = (N + 7) / 8 * 8, stage = scan_stage_elems<T, G>(N, 3);
  T* raw = reinterpret_cast<T*>(scan_sm);              // [STAGES]: x, dt, z, B rows, C rows
  // double buffers:
  float2* DU = reinterpret_cast<float2*>(raw + SCAN_STAGES * stage);  // [TT][CPB]: d, d x
  float* Bs = reinterpret_cast<float*>(DU + 2 * TT * CPB);            // [TT][NP]
  float* Cs = Bs + 2 * TT * G::NP;
  float* YP = Cs + 2 * TT * G::NP;                                    // [TT][L][YS]
  int* flags = reinterpret_cast<int*>(YP + 2 * TT * G::YT);           // first [TT], last [TT]
  const ScanBlock s = scan_block<CPB, TT>(P, blockIdx.z);
  const int tiles = s.tiles, first_t = s.tile0 * TT, segs = (P.T + SCAN_SEG - 1) / SCAN_SEG;

  if (threadIdx.x >= SCAN_MAIN) {  // tokens
    const int tid = threadIdx.x - SCAN_MAIN;
    const int pc = (tid % G::PAIRS) * 2, pt = tid / G::PAIRS;
    const float2 bias = scan_param(P.dt_bias, s, pc), skip = scan_param(P.D, s, pc);
    const RowView views[3] = {P.x, P.dt, P.z};
    ScanFetch<T, G, 3> f;
    f.init(P, s, views, tid, 3 * G::RAW, npad, s.tile0, 1);
    ScanFlags<TT> marks;
    marks.read(P, s.b, first_t, tid);
    // (both passes: all reads of shared memory, then all writes)
    constexpr int IT = TT / G::TSTEP;
    const bool spare = G::SPARE && pt >= TT;
    auto prepare = [&](int i) {
      const int t0 = first_t + i * TT, q = i & 1;
      const T* rx = raw + (i % SCAN_STAGES) * stage;
      ScanBC<T, G, 1, PAD> bc;
      float2 x[IT], dt[IT];
      float4 du[IT];
      if (!spare) {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          x[k] = scan_pair(rx + (pt + k * G::TSTEP) * CPB + pc);
          dt[k] = scan_pair(rx + G::RAW + (pt + k * G::TSTEP) * CPB + pc);
        }
      }
      bc.load(rx + 3 * G::RAW, npad, P, s, t0, tid);
      if (!spare) {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          const bool in = t0 + pt + k * G::TSTEP < P.T;
          const float d0 = scan_d(P, dt[k].x + bias.x, in), d1 = scan_d(P, dt[k].y + bias.y, in);
          du[k] = make_float4(d0, d0 * x[k].x, d1, d1 * x[k].y);
        }
#pragma unroll
        for (int k = 0; k < IT; ++k)
          *reinterpret_cast<float4*>(DU + (q * TT + pt + k * G::TSTEP) * CPB + pc) = du[k];
      }
      bc.store(Bs + q * TT * G::NP, Cs + q * TT * G::NP, tid);
      marks.write(flags + q * 2 * TT, tid);
      marks.read(P, s.b, t0 + TT, tid);
    };
    const int how = scan_how(P, s, pc);
    long long at = ((long long)s.b * P.T + first_t + pt) * P.E + s.c0 + pc;  // of the tile to finish
    const long long row_step = (long long)G::TSTEP * P.E;
    auto finish = [&](int i) {
      const int t0 = first_t + i * TT;
      const T* rx = raw + (i % SCAN_STAGES) * stage;
      const float* yp = YP + (i & 1) * TT * G::YT;
      if (spare) return;
#pragma unroll
      for (int k = 0; k < TT; k += G::TSTEP) {
        const int t = pt + k;
        const float2 x = scan_pair(rx + t * CPB + pc);
        const float2 sum = scan_join<G>(yp + t * G::YT + pc);
        float2 v = make_float2(fmaf(skip.x, x.x, sum.x), fmaf(skip.y, x.y, sum.y));
        if (P.z.p) {
          const float2 z = scan_pair(rx + 2 * G::RAW + t * CPB + pc);
          v.x *= siluf_(z.x);
          v.y *= siluf_(z.y);
        }
        if (t0 + t < P.T) scan_put_pair<T>(P.y, at, how, v);
        at += row_step;
      }
    };
    f.fetch(P, s, views, raw, first_t, tid);
    if (tiles > 1) f.fetch(P, s, views, raw + stage, first_t + TT, tid);
    cp_async_wait<0>();
    asm volatile("bar.sync 1, %0;" ::"n"(G::TOKENS) : "memory");  // the first tiles have arrived, for the whole side
    prepare(0);
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      // (stage of i + 2 held i - 2, which was finished before the last barrier)
      if (i + 2 < tiles) f.fetch(P, s, views, raw + ((i + 2) % SCAN_STAGES) * stage, first_t + (i + 2) * TT, tid);
      if (i + 1 < tiles) prepare(i + 1);
      if (i > 0) finish(i - 1);
      cp_async_wait<0>();
      __syncthreads();
    }
    finish(tiles - 1);
    return;
  }

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane / G::CH, c = warp * G::CH + lane % G::CH, n0 = l * S;
  const unsigned ok = N - n0 >= S ? (1u << S) - 1u : N > n0 ? (1u << (N - n0)) - 1u : 0u;  // states that exist
  const bool live = c < s.nc;
  Lane<S> a2 = Lane<S>::all(0.f), h = a2;
  const long long chan = (long long)(s.c0 + (live ? c : 0)) * N + n0;
#pragma unroll
  for (int i = 0; i < S; ++i)
    if (live && (ok >> i & 1)) a2.set(i, P.A[chan + i] * LOG2E);
  if (s.k > 0 && live) h = scan_enter<S, false>(P, s, chan, ok, 0);
  __syncthreads();
  for (int tile = 0; tile < tiles; ++tile) {
    const int t0 = first_t + tile * TT, q = tile & 1;
    const float2* du_ = DU + q * TT * CPB + c;
    const float* b_ = Bs + q * TT * G::NP + n0;
    const float* c_ = Cs + q * TT * G::NP + n0;
    float* y_ = YP + q * TT * G::YT + l * G::YS + c;
    const int* first = flags + q * 2 * TT;
    const int* last = first + TT;
    auto segment = [&](int t1) {
      // all of the segment's reads in front of its stores, which the compiler must assume to alias
      float2 du[SCAN_SEG];
      Lane<S> bv[SCAN_SEG], cv[SCAN_SEG];
      float y[SCAN_SEG];
#pragma unroll
      for (int k = 0; k < SCAN_SEG; ++k) {
        du[k] = du_[(t1 + k) * CPB];
        bv[k] = Lane<S>::load(b_ + (t1 + k) * G::NP);
        cv[k] = Lane<S>::load(c_ + (t1 + k) * G::NP);
      }
#pragma unroll
      for (int k = 0; k < SCAN_SEG; ++k) {
        h = lane_keep<PAD>(fma(lane_decay(a2, du[k].x), h, bv[k] * Lane<S>::all(du[k].y)), ok);
        y[k] = lane_dot(h, cv[k]);
      }
#pragma unroll
      for (int k = 0; k < SCAN_SEG; ++k) y_[(t1 + k) * G::YT] = y[k];
    };
    auto flagged = [&](int t1) {  // sequences start or end among the tokens
      const long long per = (long long)P.E * N;
#pragma unroll 1
      for (int t = t1; t < t1 + SCAN_SEG; ++t) {
        if (first[t] >= 0) h = scan_state<S>(P.h0, first[t], per, chan, live ? ok : 0u, 0);
        const float2 u = du_[t * CPB];
        h = lane_keep<PAD>(fma(lane_decay(a2, u.x), h, Lane<S>::load(b_ + t * G::NP) * Lane<S>::all(u.y)), ok);
        if (last[t] >= 0 && P.ht) {
#pragma unroll
          for (int i = 0; i < S; ++i)
            if (live && (ok >> i & 1)) P.ht[last[t] * per + chan + i] = h.get(i);
        }
        y_[t * G::YT] = lane_dot(h, Lane<S>::load(c_ + t * G::NP));
      }
    };
#pragma unroll 1
    for (int t1 = 0; t1 < TT && t0 + t1 < P.T; t1 += SCAN_SEG) {
      if (P.ckpt && live) {
        float* ck = P.ckpt + ((long long)s.b * segs + (t0 + t1) / SCAN_SEG) * P.E * N + chan;
        if (!PAD) {
          h.store(ck);
        } else {
#pragma unroll
          for (int i = 0; i < S; ++i)
            if (ok >> i & 1) ck[i] = h.get(i);
        }
      }
      if (scan_seg_flag(first + t1, last + t1)) flagged(t1);
      else segment(t1);
    }
    __syncthreads();
  }
}

template <typename T, int L, int S, bool PAD>
__global__ void __launch_bounds__(SCAN_THREADS, 2) ssm_scan_bwd_kernel(ScanParams P) {
  using G = ScanBwdGeo<T, L, S>;
  constexpr int TT = G::TT, CPB = G::CPB, CH = G::CH;
  static_assert(TT == SCAN_SEG, "a tile of the backward is one segment");
  // lane bits, from the top: XB channel bits that also order the lane's states, the L
  // lanes of a channel, the other RB channel bits (so that lane pairs share B and C reads)
  constexpr int CB = ilog2(CH), XB = CB < ilog2(S) ? CB : ilog2(S), RB = CB - XB, LB = ilog2(L);
  extern __shared__ __align__(16) char scan_sm[];
  const int N = P.N, npad = (N + 7) / 8 * 8, stage = scan_stage_elems<T, G>(N, 4);
  T* raw = reinterpret_cast<T*>(scan_sm);  // [STAGES]: x, dt, dy, z, B rows, C rows
  // three buffers (prepared, used by the recurrences, used to finish):
  float2* DU = reinterpret_cast<float2*>(raw + SCAN_STAGES * stage);  // [TT][CPB]: d, d x
  float* DS = reinterpret_cast<float*>(DU + 3 * TT * CPB);            // [TT][CPB]: dy silu(z)
  float* DZ = DS + 3 * TT * CPB;                                      // [TT][CPB]: dy silu'(z)
  // double buffers:
  float* Bs = DZ + 3 * TT * CPB;                                      // [TT][S + 1][NP]
  float* Cs = Bs + 2 * TT * G::BS;
  float* YP = Cs + 2 * TT * G::BS;           // [3][TT][L][YS]: partial sums of y, dd / ln 2, sum g B
  float* slots = YP + 2 * 3 * TT * G::YT;    // [warps][TT][2][NP]: the warps' dB and dC
  int* flags = reinterpret_cast<int*>(slots + 2 * SCAN_WARPS * TT * 2 * G::NP);  // first [TT], last [TT]
  const ScanBlock s = scan_block<CPB, TT>(P, blockIdx.z);
  const int tiles = s.tiles, tile_z = s.tile0 + tiles - 1;  // step i takes tile tile_z - i
  const int all = (P.T + TT - 1) / TT;                      // tiles of the row
  float* e = P.e_part + ((long long)s.b * P.spans + s.k) * P.E * (N + 2);

  if (threadIdx.x >= SCAN_MAIN) {  // tokens
    const int tid = threadIdx.x - SCAN_MAIN;
    const int pc = (tid % G::PAIRS) * 2, pt = tid / G::PAIRS;
    const float2 bias = scan_param(P.dt_bias, s, pc), skip = scan_param(P.D, s, pc);
    const float2 zero = make_float2(0.f, 0.f);
    // (dD_plain: what dD is where a term is infinite, of which a compensated sum makes NaN, inf - inf)
    float2 dD = zero, db = zero, dD_err = zero, db_err = zero, dD_plain = zero;
    const RowView views[4] = {P.x, P.dt, P.dy, P.z};
    ScanFetch<T, G, 4> f;
    f.init(P, s, views, tid, 4 * G::RAW, npad, tile_z, -1);
    ScanFlags<TT> marks;
    marks.read(P, s.b, tile_z * TT, tid);
    // (both passes: all reads of shared memory, then all writes)
    constexpr int IT = TT / G::TSTEP;
    const bool spare = G::SPARE && pt >= TT;
    int p3 = 0, q3 = 0;  // buffers of the next tile to prepare and to finish
    auto prepare = [&](int i) {
      const int t0 = (tile_z - i) * TT, q = i & 1;
      const T* rx = raw + (i % SCAN_STAGES) * stage;
      ScanBC<T, G, S, PAD> bc;
      float2 x[IT], dt[IT], ds[IT], z[IT];
      if (!spare) {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          const T* p = rx + (pt + k * G::TSTEP) * CPB + pc;
          x[k] = scan_pair(p);
          dt[k] = scan_pair(p + G::RAW);
          ds[k] = scan_pair(p + 2 * G::RAW);
          if (P.z.p) z[k] = scan_pair(p + 3 * G::RAW);
        }
      }
      bc.load(rx + 4 * G::RAW, npad, P, s, t0, tid);
      if (!spare) {
        const int at = (p3 * TT + pt) * CPB + pc;
        float4 du[IT];
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          const bool in = t0 + pt + k * G::TSTEP < P.T;
          const float d0 = scan_d(P, dt[k].x + bias.x, in), d1 = scan_d(P, dt[k].y + bias.y, in);
          du[k] = make_float4(d0, d0 * x[k].x, d1, d1 * x[k].y);
          if (P.z.p) {  // z becomes dy silu'(z)
            const float p0 = sigmoidf_(z[k].x), p1 = sigmoidf_(z[k].y);
            const float s0 = ds[k].x * z[k].x * p0, s1 = ds[k].y * z[k].y * p1;
            z[k] = make_float2(ds[k].x * (p0 * fmaf(z[k].x, 1.f - p0, 1.f)), ds[k].y * (p1 * fmaf(z[k].y, 1.f - p1, 1.f)));
            ds[k] = make_float2(s0, s1);
          }
        }
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          *reinterpret_cast<float4*>(DU + at + k * G::TSTEP * CPB) = du[k];
          *reinterpret_cast<float2*>(DS + at + k * G::TSTEP * CPB) = ds[k];
          if (P.z.p) *reinterpret_cast<float2*>(DZ + at + k * G::TSTEP * CPB) = z[k];
        }
      }
      p3 = p3 == 2 ? 0 : p3 + 1;
      bc.store(Bs + q * TT * G::BS, Cs + q * TT * G::BS, tid);
      marks.write(flags + q * 2 * TT, tid);
      marks.read(P, s.b, t0 - TT, tid);
    };
    const int how = scan_how(P, s, pc);
    long long to = ((long long)s.b * P.T + tile_z * TT + pt) * P.E + s.c0 + pc;  // of the tile to finish
    const long long to_step = (long long)TT * P.E, row_step = (long long)G::TSTEP * P.E;
    // the tile's dB and dC over the warps, [TT][2][N], and the step to the tile in front
    const long long part_step = (long long)P.G * P.blocks * (TT * 2 * N);
    float* part = P.bc_part + ((long long)s.b * all + tile_z) * part_step + (long long)blockIdx.x * (TT * 2 * N);
    auto finish = [&](int i) {
      const int t0 = (tile_z - i) * TT, q = i & 1, at = (q3 * TT + pt) * CPB + pc;
      q3 = q3 == 2 ? 0 : q3 + 1;
      const T* rx = raw + (i % SCAN_STAGES) * stage;
      if (!spare) {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          const int t = pt + k * G::TSTEP;
          const T* p = rx + t * CPB + pc;
          const float2 x = scan_pair(p), dt = scan_pair(p + G::RAW);
          const float4 du = *reinterpret_cast<const float4*>(DU + at + k * G::TSTEP * CPB);
          const float2 ds = *reinterpret_cast<const float2*>(DS + at + k * G::TSTEP * CPB);
          float2 dz = make_float2(0.f, 0.f);
          if (P.z.p) dz = *reinterpret_cast<const float2*>(DZ + at + k * G::TSTEP * CPB);
          const float* sums = YP + (q * 3 * TT + t) * G::YT + pc;
          const float2 s0 = scan_join<G>(sums), q0 = scan_join<G>(sums + TT * G::YT), g0 = scan_join<G>(sums + 2 * TT * G::YT);
          float2 dd = make_float2(fmaf(q0.x, LN2, g0.x * x.x), fmaf(q0.y, LN2, g0.y * x.y));
          if (P.softplus) {
            dd.x *= sigmoidf_(dt.x + bias.x);
            dd.y *= sigmoidf_(dt.y + bias.y);
          }
          if (t0 + t < P.T) {
            const long long o = to + k * row_step;
            if (P.z.p)
              scan_put_pair<T>(P.dz, o, how, make_float2(dz.x * fmaf(skip.x, x.x, s0.x), dz.y * fmaf(skip.y, x.y, s0.y)));
            scan_put_pair<T>(P.ddt, o, how, dd);
            scan_put_pair<T>(P.dx, o, how, make_float2(fmaf(g0.x, du.x, ds.x * skip.x), fmaf(g0.y, du.z, ds.y * skip.y)));
            sum_add(db.x, db_err.x, dd.x);
            sum_add(db.y, db_err.y, dd.y);
            const float2 v = make_float2(ds.x * x.x, ds.y * x.y);
            sum_add(dD.x, dD_err.x, v.x);
            sum_add(dD.y, dD_err.y, v.y);
            dD_plain.x += v.x;
            dD_plain.y += v.y;
          }
        }
      }
      const float* sl = slots + q * SCAN_WARPS * TT * 2 * G::NP;
#pragma unroll
      for (int i0 = 0; i0 < TT * 2 * G::NP; i0 += G::TOKENS) {
        const int j = i0 + tid;
        if (TT * 2 * G::NP % G::TOKENS != 0 && j >= TT * 2 * G::NP) break;
        const int n = j % G::NP;
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < SCAN_WARPS; ++w) o += sl[w * TT * 2 * G::NP + j];
        if (!PAD || n < N) part[j / G::NP * N + n] = o;
      }
      to -= to_step;
      part -= part_step;
    };
    f.fetch(P, s, views, raw, tile_z * TT, tid);
    if (tiles > 1) f.fetch(P, s, views, raw + stage, (tile_z - 1) * TT, tid);
    cp_async_wait<0>();
    asm volatile("bar.sync 1, %0;" ::"n"(G::TOKENS) : "memory");  // the first tiles have arrived, for the whole side
    prepare(0);
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      if (i + 2 < tiles) f.fetch(P, s, views, raw + ((i + 2) % SCAN_STAGES) * stage, (tile_z - 2 - i) * TT, tid);
      if (i + 1 < tiles) prepare(i + 1);
      if (i > 0) finish(i - 1);
      cp_async_wait<0>();
      __syncthreads();
    }
    finish(tiles - 1);
    // the row's dD and d dt_bias: over the side's threads of a channel pair
    asm volatile("bar.sync 1, %0;" ::"n"(G::TOKENS) : "memory");
    float4* sums = reinterpret_cast<float4*>(scan_sm);
    sums[tid] = make_float4(isnan(dD.x) ? dD_plain.x : dD.x, isnan(dD.y) ? dD_plain.y : dD.y, db.x, db.y);
    asm volatile("bar.sync 1, %0;" ::"n"(G::TOKENS) : "memory");
    if (tid < G::PAIRS) {
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = tid; k < G::TOKENS; k += G::PAIRS) {
        const float4 v = sums[k];
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
      }
      float* p = e + (long long)(s.c0 + pc) * (N + 2) + N;
      if (pc < s.nc) { p[0] = o.x; p[1] = o.z; }
      if (pc + 1 < s.nc) { p[N + 2] = o.y; p[N + 3] = o.w; }
    }
    return;
  }

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mb = lane >> (RB + LB), l = (lane >> RB) & (L - 1), ch = (mb << RB) | (lane & ((1 << RB) - 1));
  constexpr int LEFT = S >> XB;  // states of which a lane ends up with the sums
  const int m = mb * LEFT;       // register i of the lane is state n0 + (i ^ m)
  const int c = warp * CH + ch, n0 = l * S;
  const bool live = c < s.nc;
  const long long chan = (long long)(s.c0 + (live ? c : 0)) * N + n0;
  unsigned ok = 0;  // states that exist
#pragma unroll
  for (int i = 0; i < S; ++i) ok |= (unsigned)(n0 + (i ^ m) < N) << i;
  float hs[S];  // the next tile's checkpoint (left alone until then: the load is on its way)
  auto checkpoint = [&](int tile) {
    const float* p = P.ckpt + ((long long)s.b * all + tile) * P.E * N + chan;
#pragma unroll
    for (int i = 0; i < S; ++i) hs[i] = live && (!PAD || (ok >> i & 1)) ? __ldg(p + (i ^ m)) : 0.f;
  };
  checkpoint(tile_z);
  Lane<S> a2 = Lane<S>::all(0.f), r = a2;
  float dA[S], dA_err[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    dA[i] = dA_err[i] = 0.f;
    if (live && (ok >> i & 1)) a2.set(i, scan_rate(P.A[chan + (i ^ m)]));
  }
  if (s.k + 1 < P.spans && live) r = scan_enter<S, true>(P, s, chan, ok, m);
  __syncthreads();
  for (int step = 0; step < tiles; ++step) {
    const int q = step & 1, q3 = step % 3;
    const float2* du_ = DU + q3 * TT * CPB + c;
    const float* ds_ = DS + q3 * TT * CPB + c;
    const float* b_ = Bs + q * TT * G::BS + m * G::NP + n0;
    const float* c_ = Cs + q * TT * G::BS + m * G::NP + n0;
    float* y_ = YP + q * 3 * TT * G::YT + l * G::YS + c;
    float* s_ = slots + (q * SCAN_WARPS + warp) * TT * 2 * G::NP + n0;
    const int* first = flags + q * 2 * TT;
    const int* last = first + TT;
    const Lane<S> h_in = Lane<S>::of(hs);
    if (step + 1 < tiles) checkpoint(tile_z - 1 - step);

    Lane<S> dAs = Lane<S>::all(0.f);
    // Token k backwards: a, h its decay and state, `before` the state in front of it.  r leaves as what
    // passes to the token in front.
    auto token = [&](int k, const Lane<S>& a, const Lane<S>& h, const Lane<S>& before, const Lane<S>& bv,
                     const Lane<S>& cv, float2 u, float dy) {
      const Lane<S> ds = Lane<S>::all(dy);
      const Lane<S> g = lane_keep<PAD>(fma(cv, ds, r), ok);
      r = a * g;
      const Lane<S> w = lane_keep<PAD>(r * before, ok);
      dAs = fma(w, Lane<S>::all(u.x), dAs);
      const float y = lane_dot(h, cv), dd = lane_dot(w, a2), gb = lane_dot(g, bv);
      const Lane<S> vb = g * Lane<S>::all(u.y), vc = ds * h;  // dB, dC of this channel
      y_[k * G::YT] = y;
      y_[(TT + k) * G::YT] = dd;
      y_[(2 * TT + k) * G::YT] = gb;
      // over the warp's channels: states i < half stay, the others go to the lane that keeps them
      float v[2][S];
#pragma unroll
      for (int i = 0; i < S; ++i) {
        v[0][i] = vb.get(i);
        v[1][i] = vc.get(i);
      }
#pragma unroll
      for (int x = 0; x < XB; ++x) {
        const int half = S >> (x + 1);
#pragma unroll
        for (int i = 0; i < half; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b)
            v[b][i] += __shfl_xor_sync(0xffffffffu, v[b][i + half], (half / LEFT) << (RB + LB));
      }
      float* slot = s_ + k * 2 * G::NP;
      if (RB > 0) {  // one of the other channel bits decides between dB and dC, the rest just add
        const bool odd = lane & 1;
#pragma unroll
        for (int i = 0; i < LEFT; ++i) {
          const float give = odd ? v[0][i] : v[1][i], keep = odd ? v[1][i] : v[0][i];
          float o = keep + __shfl_xor_sync(0xffffffffu, give, 1);
#pragma unroll
          for (int x = 1; x < RB; ++x) o += __shfl_xor_sync(0xffffffffu, o, 1 << x);
          if ((lane & ((1 << RB) - 1)) <= 1) slot[(odd ? G::NP : 0) + (i ^ m)] = o;
        }
      } else {
#pragma unroll
        for (int i = 0; i < LEFT; ++i) {
          slot[i ^ m] = v[0][i];
          slot[G::NP + (i ^ m)] = v[1][i];
        }
      }
    };
    auto step_h = [&](const Lane<S>& a, const Lane<S>& before, const Lane<S>& bv, float2 u) {
      return lane_keep<PAD>(fma(a, before, bv * Lane<S>::all(u.y)), ok);
    };
    auto at = [&](const float* rows, int t) { return Lane<S>::load(rows + t * G::BS); };  // of B or C
    if (!scan_seg_flag(first, last)) {
      // The later half of the tokens first: its states are kept, those of the half before it only
      // passed through, and rebuilt for their own turn.  Half a segment fits the registers of two CTAs
      // per SM.  Reads come in front of stores, which the compiler must assume to alias.
      constexpr int HALF = SCAN_SEG / 2;
      Lane<S> mid = h_in;
#pragma unroll
      for (int k = 0; k < HALF; ++k) {
        const float2 u = du_[k * CPB];
        mid = step_h(lane_decay(a2, u.x), mid, at(b_, k), u);
      }
      Lane<S> h[HALF], a[HALF], bv[HALF], cv[HALF];
      float2 du[HALF];
      float dsv[HALF];
#pragma unroll
      for (int k = SCAN_SEG - 1; k >= 0; --k) {
        const int j = k % HALF;
        const Lane<S>& front = k >= HALF ? mid : h_in;  // the state in front of the half
        if (j == HALF - 1) {
#pragma unroll
          for (int o = 0; o < HALF; ++o) {
            const int t = k - HALF + 1 + o;
            du[o] = du_[t * CPB];
            dsv[o] = ds_[t * CPB];
            bv[o] = at(b_, t);
            cv[o] = at(c_, t);
          }
#pragma unroll
          for (int o = 0; o < HALF; ++o) {
            a[o] = lane_decay(a2, du[o].x);
            h[o] = step_h(a[o], o ? h[o ? o - 1 : 0] : front, bv[o], du[o]);
          }
        }
        token(k, a[j], h[j], j ? h[j ? j - 1 : 0] : front, bv[j], cv[j], du[j], dsv[j]);
      }
    } else {
      // a sequence starts or ends here: token by token, the states in front of them kept in local memory
      const long long per = (long long)P.E * N;
      Lane<S> front[SCAN_SEG], h = h_in;
#pragma unroll 1
      for (int k = 0; k < SCAN_SEG; ++k) {
        if (first[k] >= 0) h = scan_state<S>(P.h0, first[k], per, chan, live ? ok : 0u, m);
        front[k] = h;
        const float2 u = du_[k * CPB];
        h = step_h(lane_decay(a2, u.x), h, at(b_, k), u);
      }
#pragma unroll 1
      for (int k = SCAN_SEG - 1; k >= 0; --k) {
        if (last[k] >= 0) r = r + scan_state<S>(P.dht, last[k], per, chan, live ? ok : 0u, m);
        const float2 u = du_[k * CPB];
        const Lane<S> a = lane_decay(a2, u.x), bv = at(b_, k), before = front[k];
        token(k, a, step_h(a, before, bv, u), before, bv, at(c_, k), u, ds_[k * CPB]);
        if (first[k] >= 0) {  // what reaches the initial state; nothing passes the start
          if (P.dh0 && live) {
#pragma unroll
            for (int i = 0; i < S; ++i)
              if (ok >> i & 1) P.dh0[first[k] * per + chan + (i ^ m)] = r.get(i);
          }
          r = Lane<S>::all(0.f);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < S; ++i) sum_add(dA[i], dA_err[i], dAs.get(i));
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < S; ++i)
    if (live && (ok >> i & 1)) e[(long long)(s.c0 + c) * (N + 2) + n0 + (i ^ m)] = dA[i];
}

// dB and dC: the channel blocks' partial sums of a tile ([TT][2][N]), summed in block
// order.  One CTA column per (row, tile, group).
constexpr int SCAN_BC_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(SCAN_BC_THREADS) ssm_scan_bc_kernel(const float* part, int T_, int tiles, int Gr,
                                                                      int blocks, int N, T* dB, T* dC) {
  const int per = SCAN_TT_BWD * 2 * N;
  const int i = blockIdx.y * SCAN_BC_THREADS + threadIdx.x;
  if (i >= per) return;
  const long long w = blockIdx.x;  // (row, tile, group)
  const float* p = part + w * blocks * (long long)per + i;
  float acc = 0.f;
#pragma unroll 8
  for (int k = 0; k < blocks; ++k) acc += p[(long long)k * per];
  const int t = i / (2 * N), rest = i - t * 2 * N, half = rest >= N, n = rest - half * N;
  const int g = (int)(w % Gr);
  const long long bt = w / Gr;
  const int tok = (int)(bt % tiles) * SCAN_TT_BWD + t;
  if (tok < T_) (half ? dC : dB)[(((bt / tiles) * T_ + tok) * Gr + g) * N + n] = io_from_f<T>(acc);
}

// One token for each of `rows` requests: the slot's state [E][N] is read, stepped
// and rewritten; every other input is a row.  Memory bound on the states.  A state's arithmetic is the scan's,
// operation by operation (lane_decay's centred exponential too): decoded token by token it has the bits that a
// prompt of one span gives it.
// A thread owns 4 Q states of a channel (LP lanes per channel, y summed by shuffles) and
// walks the rows with its A in registers; the grid is twice what the GPU holds.  Eight states
// a thread rather than four halve the work per state on softplus and addresses, which
// bounded it: 512 rows x 2048 channels x 16 states, bf16, states not in the L2: 29.6 us (4.8 TB/s) against
// 43 us; 36 us with registers for 3 or 5 CTAs per SM.
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

template <typename T, int LP, int Q, bool VEC>
__global__ void __launch_bounds__(STEP_THREADS, 4) ssm_scan_step_kernel(ScanStepParams P) {
  constexpr int S = 4 * Q;
  const long long idx = (long long)blockIdx.x * STEP_THREADS + threadIdx.x;
  const int e = (int)(idx / LP), n0 = (int)(idx % LP) * 4, N = P.N;  // states n0 + 4 LP q + k, q < Q, k < 4
  const bool ok = e < P.E;  // (whole channels: the shuffles below stay inside one)
  const int ec = ok ? e : 0, g = ec / (P.E / P.G), step = gridDim.y, per = P.E * N;
  auto at = [&](int i) { return i / 4 * 4 * LP + i % 4; };  // state n0 + at(i) is the thread's i-th
  float* const states = P.state + (long long)ec * N + n0;
  // addresses of a row's inputs and the steps to the next (added up, not multiplied: the kernel issues less)
  int r = blockIdx.y;
  const T* px = static_cast<const T*>(P.x) + r * P.sx + ec;
  const T* pdt = static_cast<const T*>(P.dt) + r * P.sdt + ec;
  const T* pz = static_cast<const T*>(P.z) + r * P.sz + ec;
  const T* pB = static_cast<const T*>(P.Bm) + r * P.b_sb + g * P.b_sg + n0;
  const T* pC = static_cast<const T*>(P.Cm) + r * P.c_sb + g * P.c_sg + n0;
  T* py = static_cast<T*>(P.y) + (long long)r * P.E + ec;
  const long long dx = step * P.sx, ddt = step * P.sdt, dz = step * P.sz, dB = step * P.b_sb, dC = step * P.c_sb,
                  dy = (long long)step * P.E;
  int s = step_slot(P.slots, r, P.pool, P.err);
  float a[S];
#pragma unroll
  for (int i = 0; i < S; ++i) a[i] = n0 + at(i) < N ? __ldg(P.A + (long long)ec * N + n0 + at(i)) * LOG2E : 0.f;
  const float D = P.D ? __ldg(P.D + ec) : 0.f, bias = P.dt_bias ? __ldg(P.dt_bias + ec) : 0.f;
  while (true) {
    const int after = r + step < P.rows ? step_slot(P.slots, r + step, P.pool, P.err) : -1;
    float y = 0.f, x = 0.f, z = 0.f;
    if (s >= 0 && ok) {
      float* st = states + (long long)s * per;
      float h[S];
      IoVec<T, 4> B[Q], C[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int o = 4 * LP * q;
        if (VEC) {
          if (n0 + o < N) {
            const float4 v = *reinterpret_cast<const float4*>(st + o);
            h[4 * q] = v.x; h[4 * q + 1] = v.y; h[4 * q + 2] = v.z; h[4 * q + 3] = v.w;
            B[q] = *reinterpret_cast<const IoVec<T, 4>*>(pB + o);
            C[q] = *reinterpret_cast<const IoVec<T, 4>*>(pC + o);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n0 + o + k < N) {
              h[4 * q + k] = st[o + k];
              B[q].v[k] = pB[o + k];
              C[q].v[k] = pC[o + k];
            }
        }
      }
      x = io_to_f(*px);
      float d = io_to_f(*pdt) + bias;
      if (P.z && n0 == 0) z = io_to_f(*pz);
      if (P.softplus) d = softplusf_(d);
      const float u = d * x;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int o = 4 * LP * q;
        if (VEC && n0 + o >= N) continue;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (VEC || n0 + o + k < N) {
            float& v = h[4 * q + k];
            v = fmaf(ex2(fmaf(a[4 * q + k], d, SCAN_EXP_SHIFT)), v, u * io_to_f(B[q].v[k]));
            y = fmaf(v, io_to_f(C[q].v[k]), y);
            if (!VEC) st[o + k] = v;
          }
        if (VEC) *reinterpret_cast<float4*>(st + o) = make_float4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]);
      }
    }
#pragma unroll
    for (int m = LP / 2; m >= 1; m >>= 1) y += __shfl_xor_sync(0xffffffffu, y, m);
    if (ok && n0 == 0) {
      y = fmaf(D, x, y);
      if (P.z) y *= siluf_(z);
      *py = io_from_f<T>(s >= 0 ? y : 0.f);
    }
    r += step;
    if (r >= P.rows) break;
    px += dx;
    pdt += ddt;
    pz += dz;
    pB += dB;
    pC += dC;
    py += dy;
    s = after;
  }
}

}  // namespace kda
