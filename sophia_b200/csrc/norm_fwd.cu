// The residual norm's forward kernels.
#include "norm_launch.cuh"

namespace kda {

template <typename TX, typename TO>
int rn_fwd(RnParams& p, bool vec, cudaStream_t st) {
  if (vec) {
    constexpr int HALF = 8 * sizeof(TO) / 16;  // pieces of a thread with 8 channels
    const RnShape s = rn_ring_shape(p.D, sizeof(TO));
    const RnFit fit = rn_fwd_fit<TX, TO>(p, s);
    p.warps = s.warps;
    p.lanes = s.lanes;
    if (fit.stages > 0)
      return s.k == HALF ? launch_rn_fwd_ring<TX, TO, HALF>(p, s, fit, st) : launch_rn_fwd_ring<TX, TO, 2 * HALF>(p, s, fit, st);
  }
  const RnShape s = rn_plain_shape(p.D);
  p.warps = s.warps;
  if (s.k == 2) return launch_rn_fwd<TX, TO, 2>(p, s, st);
  if (s.k == 4) return launch_rn_fwd<TX, TO, 4>(p, s, st);
  return launch_rn_fwd<TX, TO, 16>(p, s, st);
}

template int rn_fwd<float, float>(RnParams&, bool, cudaStream_t);
template int rn_fwd<bf16, bf16>(RnParams&, bool, cudaStream_t);
template int rn_fwd<f16, f16>(RnParams&, bool, cudaStream_t);
template int rn_fwd<float, bf16>(RnParams&, bool, cudaStream_t);
template int rn_fwd<float, f16>(RnParams&, bool, cudaStream_t);

}  // namespace kda
