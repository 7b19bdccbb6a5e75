// The residual norm's forward, for one pair of types a translation unit (norm_fwd_*.cu).
#pragma once

#include "norm_launch.cuh"

namespace kda {

template <typename TX, typename TO, int K, bool NARROW>
struct RnForward {
  template <bool FULL, bool GATE, bool DROP>
  static auto get() { return rn_fwd_ring_kernel<TX, TO, K, NARROW, FULL && !NARROW, GATE, DROP>; }
};

template <typename TX, typename TO>
int rn_fwd(RnParams& p, bool vec, cudaStream_t st) {
  if (vec && p.rows <= INT32_MAX / 2) {
    const RnShape s = rn_fwd_shape(p.D, sizeof(TO));
    const RnFit fit = rn_fwd_fit<TX, TO>(p, s);
    p.warps = s.warps;
    p.lanes = s.lanes;
    if (fit.stages > 0) {
      constexpr int V = 16 / sizeof(TO);
      const char* what = "residual norm forward";
      if (p.D <= 256) return launch_rn_ring<RnForward<TX, TO, 8 / V, true>>(p, s, fit, K_NORM_FWD, what, st);
      if (s.k == 16 / V) return launch_rn_ring<RnForward<TX, TO, 16 / V, false>>(p, s, fit, K_NORM_FWD, what, st);
      if (s.k == 24 / V) return launch_rn_ring<RnForward<TX, TO, 24 / V, false>>(p, s, fit, K_NORM_FWD, what, st);
      return launch_rn_ring<RnForward<TX, TO, 32 / V, false>>(p, s, fit, K_NORM_FWD, what, st);
    }
  }
  const RnShape s = rn_plain_shape(p.D);
  p.warps = s.warps;
  if (s.k == 2) return launch_rn_fwd<TX, TO, 2>(p, s, st);
  return launch_rn_fwd<TX, TO, 4>(p, s, st);
}

}  // namespace kda
