// Shapes and launches of the selective scan's kernels.  The kernels are
// instantiated per activation type in a translation unit of their own.
#pragma once

#include <algorithm>
#include <string>

#include "kda_host.h"
#include "ssm_scan.cuh"

namespace kda {

struct ScanGrads {  // outputs of the backward's reductions
  float *dA, *dD, *ddt_bias;
  void *dB, *dC;
};
template <typename T> int scan_fwd(const ScanParams& p, cudaStream_t st);
template <typename T> int scan_bwd(const ScanParams& p, const ScanGrads& g, cudaStream_t st);

// States per lane.  Four do the most work per value read from shared memory and per token that is
// passed between the two sides; two give twice the CTAs, but spans give more of them for less (1 x 8192
// tokens x 2048 channels, N = 16: forward and backward 374 + 1147 us with two states, one span).
constexpr int SCAN_S = 4;

// Lanes per channel.
inline int scan_lanes(int N) {
  int l = 2;
  while (l * SCAN_S < N) l <<= 1;
  return l;
}
inline int scan_blocks(int E, int G, int L) {
  const int cpb = SCAN_WARPS * (32 / L);
  return (E / G + cpb - 1) / cpb;
}
// How a pass is cut: spans of `span` tokens, forward tiles of `tile` tokens.
struct ScanCut {
  int span, tile;
  int spans(long long T) const { return (int)((T + span - 1) / span); }
};
// Of the numbers k of spans (and of the tiles) the one that costs least, in tokens of a CTA of the scan that shares
// its SM with another.  An SM takes its CTAs two at a time, three at a time in the carries' kernel, one at a time
// in the backward of more than 40 states (fp32: more than 32; 117 KB of shared memory and more).  A lone CTA takes
// 0.68 (up to 8 states: 0.83; more than 56 in 16 bits: 0.81; in the carries' kernel 0.5, two 0.71) of a full SM's time;
// the carries' token costs 1.04 of the forward's, 0.37 of the backward's (0.081 us of 0.078 and 0.217, measured:
// bf16, N = 16; 0.24 of 0.34 us for the backward's lone CTA of 64 states).  Up to 8 states forward, rows in 16-byte
// pieces: 0.66 of 0.117 us, there a lone CTA 0.75, two 0.8 (3 x 8021 x 2520 tokens and channels in 4, 6, 8, 12 spans:
// 645, 656, 648, 590 us by this, 669, 661, 634, 591 measured).  A CTA's start and a launch count 40 tokens each,
// composing a span's carry half a token of every CTA, on average.
//
// Tiles of the forward: 32 tokens in 16 bits, 16 in fp32 (two CTAs of 32 would not fit an SM).  In 16 bits two CTAs
// of 32 do not fit either with up to 8 states (64 channels a CTA) and with more than 56 (rows of B and C).  There 16
// tokens bring the second CTA, and 32 are the faster for one alone: 0.69 and 0.67 of a full SM's time.  So 32 where
// the grid gives no SM a second one, from 64 tokens on (one CTA per SM, 3 states, us with 16 and with 32: 16 tokens
// 10.2 and 11.0, 33 tokens 13.2 and 13.2, 64 tokens 15.3 and 13.3); with up to 8 states only where rows are read in
// 16-byte pieces (element by element, 120 x 2048 x 61: 429 us with 16 and spans, 609 with 32).  Measured, bf16, 8 and 64
// states, us with 16 and with 32 (one span): one CTA per SM, 148 x 2048 tokens, 207 and 170, 141 and 117; two, 240
// and 334, 174 and 226.  4 x 4096 x 2048, 8 states: 343 (four spans) and 330.
inline ScanCut scan_cut(long long B, long long T, int E, int N, int G, bool half, bool vec, bool backward) {
  const int L = scan_lanes(N);
  const long long ctas = B * G * scan_blocks(E, G, L);
  const int sms = sm_count();
  const bool one = backward && N > (half ? 40 : 32);
  const bool few = !backward && L == 2 && vec;
  const bool pick = half && !backward && (L == 2 || N > 56);  // the tiles are chosen by the grid
  const float weight = backward ? (one ? 0.24f : 0.37f) : few ? 0.66f : 1.04f;
  const float lone = L == 2 ? 0.83f : pick ? 0.81f : 0.68f, lone32 = few ? 0.69f : 0.67f;
  auto two = [&](long long n) { return one ? (float)n : (float)(n / 2) + (n % 2 ? lone : 0.f); };
  const float carry1 = few ? 0.75f : 0.5f, carry2 = few ? 0.8f : 0.71f;
  auto three = [&](long long n) { return (float)(n / 3) + (n % 3 == 2 ? carry2 : n % 3 ? carry1 : 0.f); };
  ScanCut best{(int)T, 16};
  float least = 0.f;
  const long long most = std::min<long long>(64, T / 64);
  for (long long k = 1; k == 1 || k <= most; ++k) {
    const long long span = ((T + k - 1) / k + 31) / 32 * 32;
    if (k > 1 && (T + span - 1) / span != k) continue;
    const float t = (float)span + 40.f;
    const bool wide = half && (!pick || ((few || N > 56) && ctas * k <= sms && T >= 64));
    const float per_sm = pick && wide ? lone32 : two((ctas * k + sms - 1) / sms);
    const float cost = per_sm * (t + 0.5f * k) +
                       (k > 1 ? three((ctas * (k - 1) + sms - 1) / sms) * weight * t + 40.f : 0.f);
    if (k == 1 || cost < least) {
      least = cost;
      best = {(int)span, wide ? 32 : 16};
    }
  }
  return best;
}
// The most spans that a pass of any type and alignment is cut into (its workspace has room for them).
inline int scan_most_spans(long long B, long long T, int E, int N, int G, bool backward) {
  auto spans = [&](bool half, bool vec) { return scan_cut(B, T, E, N, G, half, vec, backward).spans(T); };
  int n = spans(true, true);
  if (backward ? N > 32 && N <= 40 : N <= 8 || N > 56) n = std::max(n, spans(false, true));
  if (!backward && N <= 8) n = std::max(n, spans(false, false));  // (as in 16 bits)
  return n;
}
// Bytes of the spans' carries (none for one span).
inline size_t scan_carry_bytes(long long B, int spans, int E, int N) {
  return spans > 1 ? (size_t)B * spans * E * N * 8 : 0;
}
// Floats of the backward's dB / dC partial sums.
inline long long scan_part_floats(long long B, long long T, int E, int N, int G) {
  return B * ((T + SCAN_TT_BWD - 1) / SCAN_TT_BWD) * G * scan_blocks(E, G, scan_lanes(N)) * SCAN_TT_BWD * 2 * N;
}

#ifdef SSM_SCAN_INSTANTIATE
// Sets a kernel's shared-memory limit to what its most states need: the same for every call, because host threads with
// fewer states may be here too.
template <typename K>
int scan_limit(K kernel, int most, const char* what) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  return e == cudaSuccess ? KDA_OK : fail(KDA_ERR_CUDA, std::string(what) + " smem: " + cudaGetErrorString(e));
}
// P and c of the spans, if there are several.
template <typename T, int L, bool PAD, bool REV>
int launch_scan_carry(const ScanParams& p, cudaStream_t st) {
  if (p.spans == 1) return KDA_OK;
  auto bytes = [](int N) { return scan_carry_smem<T, ScanCarryGeo<T, L, SCAN_S>>(N, REV ? 3 : 2); };
  const int smem = bytes(p.N);
  auto kernel = ssm_scan_carry_kernel<T, L, SCAN_S, PAD, REV>;
  if (int rc = scan_limit(kernel, bytes(L * SCAN_S), "scan carry")) return rc;
  {
    TimedLaunch tl(REV ? K_SCAN_BWD : K_SCAN_FWD, st);
    kernel<<<dim3(p.G * p.blocks, p.B, p.spans - 1), SCAN_THREADS, smem, st>>>(p);
  }
  return launch_check("scan carry");
}

template <typename T, int L, int TT, bool PAD>
int launch_scan_fwd_tile(const ScanParams& p, cudaStream_t st) {
  constexpr int S = SCAN_S;
  using G = ScanGeo<T, L, S, TT>;
  const int smem = scan_fwd_smem<T, G>(p.N);
  auto kernel = ssm_scan_fwd_kernel<T, L, S, TT, PAD>;
  if (int rc = scan_limit(kernel, scan_fwd_smem<T, G>(L * S), "scan forward")) return rc;
  {
    TimedLaunch tl(K_SCAN_FWD, st);
    kernel<<<dim3(p.G * p.blocks, p.B, p.spans), SCAN_THREADS, smem, st>>>(p);
  }
  return launch_check("scan forward");
}

template <typename T, int L, bool PAD>
int launch_scan_fwd(ScanParams p, cudaStream_t st) {
  p.blocks = scan_blocks(p.E, p.G, L);
  const int rc = launch_scan_carry<T, L, PAD, false>(p, st);
  if (rc) return rc;
  if constexpr (sizeof(T) == 4) return launch_scan_fwd_tile<T, L, 16, PAD>(p, st);
  else if constexpr (L == 2 || L == 16)
    return p.tile == 32 ? launch_scan_fwd_tile<T, L, 32, PAD>(p, st) : launch_scan_fwd_tile<T, L, 16, PAD>(p, st);
  else return launch_scan_fwd_tile<T, L, 32, PAD>(p, st);
}

template <typename T, int L, bool PAD>
int launch_scan_bwd(ScanParams p, const ScanGrads& g, cudaStream_t st) {
  constexpr int S = SCAN_S;
  using G = ScanBwdGeo<T, L, S>;
  p.blocks = scan_blocks(p.E, p.G, L);
  if (int rc = launch_scan_carry<T, L, PAD, true>(p, st)) return rc;
  const int smem = scan_bwd_smem<T, G>(p.N);
  auto kernel = ssm_scan_bwd_kernel<T, L, S, PAD>;
  if (int rc = scan_limit(kernel, scan_bwd_smem<T, G>(L * S), "scan backward")) return rc;
  const int tiles = (p.T + G::TT - 1) / G::TT, per = G::TT * 2 * p.N;
  const long long cols = (long long)p.E * (p.N + 2);
  {
    TimedLaunch tl(K_SCAN_BWD, st);
    kernel<<<dim3(p.G * p.blocks, p.B, p.spans), SCAN_THREADS, smem, st>>>(p);
    ssm_scan_bc_kernel<T><<<dim3((unsigned)((long long)p.B * tiles * p.G), (per + SCAN_BC_THREADS - 1) / SCAN_BC_THREADS),
                            SCAN_BC_THREADS, 0, st>>>(p.bc_part, p.T, tiles, p.G, p.blocks, p.N, static_cast<T*>(g.dB),
                                                      static_cast<T*>(g.dC));
    ssm_reduce_kernel<<<(unsigned)((cols + SSM_REDUCE_COLS - 1) / SSM_REDUCE_COLS), SSM_REDUCE_COLS * SSM_REDUCE_SLICES,
                        0, st>>>(p.e_part, (long long)p.B * p.spans, cols, p.N, p.N + 2, g.dA, g.dD, g.ddt_bias);
  }
  return launch_check("scan backward");
}

template <typename T>
int scan_fwd(const ScanParams& p, cudaStream_t st) {
  const int L = scan_lanes(p.N);
  const bool pad = p.N != L * SCAN_S;
#define SCAN_CASE(l) \
  if (L == l) return pad ? launch_scan_fwd<T, l, true>(p, st) : launch_scan_fwd<T, l, false>(p, st);
  SCAN_CASE(2) SCAN_CASE(4) SCAN_CASE(8) SCAN_CASE(16)
#undef SCAN_CASE
  return fail(KDA_ERR_UNSUPPORTED, "no scan kernel for this state size");
}
template <typename T>
int scan_bwd(const ScanParams& p, const ScanGrads& g, cudaStream_t st) {
  const int L = scan_lanes(p.N);
  const bool pad = p.N != L * SCAN_S;
#define SCAN_CASE(l) \
  if (L == l) return pad ? launch_scan_bwd<T, l, true>(p, g, st) : launch_scan_bwd<T, l, false>(p, g, st);
  SCAN_CASE(2) SCAN_CASE(4) SCAN_CASE(8) SCAN_CASE(16)
#undef SCAN_CASE
  return fail(KDA_ERR_UNSUPPORTED, "no scan kernel for this state size");
}
template int scan_fwd<SSM_SCAN_INSTANTIATE>(const ScanParams&, cudaStream_t);
template int scan_bwd<SSM_SCAN_INSTANTIATE>(const ScanParams&, const ScanGrads&, cudaStream_t);
#endif

}  // namespace kda
