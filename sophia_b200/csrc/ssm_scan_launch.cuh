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

// Lanes per channel for S states a lane.
inline int scan_lanes(int N, int S) {
  int l = S == 4 ? 2 : 4;
  while (l * S < N) l <<= 1;
  return l;
}
inline int scan_blocks(int E, int G, int L) {
  const int cpb = SCAN_WARPS * (32 / L);
  return (E / G + cpb - 1) / cpb;
}
// States per lane.  Four keep the most work per value read from shared memory; where they
// leave more than half of the SMs without a CTA, two make twice the CTAs.  Measured (bf16, N = 16,
// forward and backward, us): 4 x 4096 tokens x 2048 channels (256 CTAs of four states) 319 + 992
// against 527 + 1537 with two; 1 x 8192 x 2048 (64 CTAs) 450 + 1453 against 377 + 1211.
// More than 32 states run with four in any case.
inline int scan_states(long long B, int E, int N, int G) {
  if (N > 32) return 4;
  return 2 * B * G * scan_blocks(E, G, scan_lanes(N, 4)) >= sm_count() ? 4 : 2;
}
// Floats of the backward's dB / dC partial sums.
inline long long scan_part_floats(long long B, long long T, int E, int N, int G) {
  const int L = scan_lanes(N, scan_states(B, E, N, G));
  return B * ((T + SCAN_TT_BWD - 1) / SCAN_TT_BWD) * G * scan_blocks(E, G, L) * SCAN_TT_BWD * 2 * N;
}

#ifdef SSM_SCAN_INSTANTIATE
template <typename T, int L, int S, bool PAD>
int launch_scan_fwd(ScanParams p, cudaStream_t st) {
  using G = ScanFwdGeo<T, L, S>;
  p.blocks = scan_blocks(p.E, p.G, L);
  const int smem = scan_fwd_smem<T, G>(p.N);
  auto kernel = ssm_scan_fwd_kernel<T, L, S, PAD>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return fail(KDA_ERR_CUDA, std::string("scan forward smem: ") + cudaGetErrorString(e));
  {
    TimedLaunch tl(K_SCAN_FWD, st);
    kernel<<<dim3(p.G * p.blocks, p.B), SCAN_THREADS, smem, st>>>(p);
  }
  return launch_check("scan forward");
}

template <typename T, int L, int S, bool PAD>
int launch_scan_bwd(ScanParams p, const ScanGrads& g, cudaStream_t st) {
  using G = ScanBwdGeo<T, L, S>;
  p.blocks = scan_blocks(p.E, p.G, L);
  const int smem = scan_bwd_smem<T, G>(p.N);
  auto kernel = ssm_scan_bwd_kernel<T, L, S, PAD>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return fail(KDA_ERR_CUDA, std::string("scan backward smem: ") + cudaGetErrorString(e));
  const int tiles = (p.T + G::TT - 1) / G::TT, per = G::TT * 2 * p.N;
  const long long cols = (long long)p.E * (p.N + 2);
  {
    TimedLaunch tl(K_SCAN_BWD, st);
    kernel<<<dim3(p.G * p.blocks, p.B), SCAN_THREADS, smem, st>>>(p);
    ssm_scan_bc_kernel<T><<<dim3((unsigned)((long long)p.B * tiles * p.G), (per + SCAN_BC_THREADS - 1) / SCAN_BC_THREADS),
                            SCAN_BC_THREADS, 0, st>>>(p.bc_part, p.T, tiles, p.G, p.blocks, p.N, static_cast<T*>(g.dB),
                                                      static_cast<T*>(g.dC));
    ssm_reduce_kernel<<<(unsigned)((cols + SSM_REDUCE_COLS - 1) / SSM_REDUCE_COLS), SSM_REDUCE_COLS * SSM_REDUCE_SLICES,
                        0, st>>>(p.e_part, p.B, cols, p.N, p.N + 2, g.dA, g.dD, g.ddt_bias);
  }
  return launch_check("scan backward");
}

template <typename T>
int scan_fwd(const ScanParams& p, cudaStream_t st) {
  const int S = scan_states(p.B, p.E, p.N, p.G), L = scan_lanes(p.N, S);
  const bool pad = p.N != L * S;
#define SCAN_CASE(l, s) \
  if (L == l && S == s) return pad ? launch_scan_fwd<T, l, s, true>(p, st) : launch_scan_fwd<T, l, s, false>(p, st);
  SCAN_CASE(2, 4) SCAN_CASE(4, 4) SCAN_CASE(8, 4) SCAN_CASE(16, 4)
  SCAN_CASE(4, 2) SCAN_CASE(8, 2) SCAN_CASE(16, 2)
#undef SCAN_CASE
  return fail(KDA_ERR_UNSUPPORTED, "no scan kernel for this state size");
}
template <typename T>
int scan_bwd(const ScanParams& p, const ScanGrads& g, cudaStream_t st) {
  const int S = scan_states(p.B, p.E, p.N, p.G), L = scan_lanes(p.N, S);
  const bool pad = p.N != L * S;
#define SCAN_CASE(l, s) \
  if (L == l && S == s) return pad ? launch_scan_bwd<T, l, s, true>(p, g, st) : launch_scan_bwd<T, l, s, false>(p, g, st);
  SCAN_CASE(2, 4) SCAN_CASE(4, 4) SCAN_CASE(8, 4) SCAN_CASE(16, 4)
  SCAN_CASE(4, 2) SCAN_CASE(8, 2) SCAN_CASE(16, 2)
#undef SCAN_CASE
  return fail(KDA_ERR_UNSUPPORTED, "no scan kernel for this state size");
}
template int scan_fwd<SSM_SCAN_INSTANTIATE>(const ScanParams&, cudaStream_t);
template int scan_bwd<SSM_SCAN_INSTANTIATE>(const ScanParams&, const ScanGrads&, cudaStream_t);
#endif

}  // namespace kda
