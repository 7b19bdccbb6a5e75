// Shapes and launches of the residual norm's kernels, shared by the translation units of its two directions.
#pragma once

#include <algorithm>
#include <string>

#include "kda_host.h"
#include "residual_norm.cuh"

namespace kda {

// How a row is laid over threads: `warps` of a group, k pieces of v channels a thread, groups of a CTA.
struct RnShape {
  int v, k, warps, groups;
};
// Whole pieces (16 bytes of the branch's type) wherever rows are aligned to them, else single channels.  Backward as few
// pieces a thread as 16 warps allow: its registers hold five tensors.
inline RnShape rn_shape(int D, size_t branch_size, bool vec, bool backward) {
  RnShape s;
  s.v = vec ? (int)(16 / branch_size) : 1;
  const int pieces = (D + s.v - 1) / s.v;
  if (vec) {
    s.k = 1;
    while (pieces > 32 * s.k * (backward ? RN_MAX_WARPS : 8)) s.k *= 2;
    if (s.k > 4) s.k = 4;
  } else {
    s.k = pieces <= 64 * 8 ? 2 : (pieces <= 32 * 4 * RN_MAX_WARPS ? 4 : 16);
  }
  s.warps = (pieces + 32 * s.k - 1) / (32 * s.k);
  s.groups = std::max(1, 8 / s.warps);
  return s;
}
inline int rn_bwd_ctas(const RnShape& s) { return std::max(1, 24 / (s.warps * s.groups)); }  // per SM
inline long long rn_bwd_grid(long long rows, const RnShape& s) {
  return std::max(1LL, std::min((rows + s.groups - 1) / s.groups, (long long)rn_bwd_ctas(s) * sm_count()));
}

template <typename TX, typename TO>
int rn_fwd(RnParams& p, bool vec, cudaStream_t st);
template <typename TX, typename TO>
int rn_bwd(RnParams& p, bool vec, cudaStream_t st);

template <typename TX, typename TO, int V, int K>
int launch_rn_fwd(const RnParams& p, const RnShape& s, cudaStream_t st) {
  const long long ctas = (p.rows + s.groups - 1) / s.groups;
  {
    TimedLaunch tl(K_NORM_FWD, st);
    rn_fwd_kernel<TX, TO, V, K>
        <<<(unsigned)std::min(ctas, 1LL << 20), s.warps * s.groups * 32, 0, st>>>(p);
  }
  return launch_check("residual norm forward");
}

template <typename TX, typename TO, int V, int K>
int launch_rn_bwd(const RnParams& p, const RnShape& s, cudaStream_t st) {
  const size_t smem = (size_t)s.groups * 3 * p.D * 4;
  auto kernel = rn_bwd_kernel<TX, TO, V, K>;
  if (smem > 40 * 1024) {  // (48 KB go without asking, the static ones included)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return fail(KDA_ERR_CUDA, std::string("residual norm smem: ") + cudaGetErrorString(e));
  }
  {
    TimedLaunch tl(K_NORM_BWD, st);
    kernel<<<(unsigned)rn_bwd_grid(p.rows, s), s.warps * s.groups * 32, smem, st>>>(p);
  }
  return launch_check("residual norm backward");
}

}  // namespace kda
