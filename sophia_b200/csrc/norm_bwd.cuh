// The residual norm's backward, for one pair of types a translation unit (norm_bwd_*.cu).
#pragma once

#include "norm_launch.cuh"

namespace kda {

template <typename TX, typename TO, bool NARROW>
struct RnBackward {
  template <bool FULL, bool GATE, bool DROP>
  static auto get() { return rn_bwd_ring_kernel<TX, TO, NARROW, FULL && !NARROW, GATE, DROP>; }
};

template <typename TX, typename TO>
int rn_bwd(RnParams& p, bool vec, cudaStream_t st) {
  if (vec && p.rows <= INT32_MAX / 2) {
    const RnShape s = rn_bwd_shape(p.D, sizeof(TO));
    const RnFit fit = rn_bwd_fit<TX, TO>(p, s);
    p.warps = s.warps;
    p.lanes = s.lanes;
    if (fit.stages > 0) {
      const char* what = "residual norm backward";
      if (p.D <= 256) return launch_rn_ring<RnBackward<TX, TO, true>>(p, s, fit, K_NORM_BWD, what, st);
      return launch_rn_ring<RnBackward<TX, TO, false>>(p, s, fit, K_NORM_BWD, what, st);
    }
  }
  const RnShape s = rn_plain_shape(p.D);
  p.warps = s.warps;
  if (s.k == 2) return launch_rn_bwd<TX, TO, 2>(p, s, st);
  return launch_rn_bwd<TX, TO, 4>(p, s, st);
}

}  // namespace kda
