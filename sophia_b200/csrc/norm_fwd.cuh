// The residual norm's forward, for one pair of types a translation unit (norm_fwd_*.cu).
#pragma once

#include "norm_launch.cuh"

namespace kda {

template <typename TX, typename TO, bool NARROW, bool FULL, bool GATE, bool DROP>
struct RnForward {
  static auto get() { return rn_fwd_ring_kernel<TX, TO, NARROW, FULL, GATE, DROP>; }
};

template <typename TX, typename TO>
int rn_fwd(RnParams& p, bool vec, cudaStream_t st) {
  if (vec && p.rows <= INT32_MAX / 2) {
    const RnShape s = rn_ring_shape(p.D, sizeof(TO));
    const RnFit fit = rn_fwd_fit<TX, TO>(p, s);
    p.warps = s.warps;
    p.lanes = s.lanes;
    if (fit.stages > 0) return launch_rn_ring<RnForward, TX, TO>(p, s, fit, K_NORM_FWD, "residual norm forward", st);
  }
  const RnShape s = rn_plain_shape(p.D);
  p.warps = s.warps;
  if (s.k == 2) return launch_rn_fwd<TX, TO, 2>(p, s, st);
  if (s.k == 4) return launch_rn_fwd<TX, TO, 4>(p, s, st);
  return launch_rn_fwd<TX, TO, 16>(p, s, st);
}

}  // namespace kda
