// The residual norm's backward kernels.
#include "norm_launch.cuh"

namespace kda {

template <typename TX, typename TO>
int rn_bwd(RnParams& p, bool vec, cudaStream_t st) {
  const RnShape s = rn_shape(p.D, sizeof(TO), vec, true);
  constexpr int V = 16 / sizeof(TO);
  p.warps = s.warps;
  if (vec) {
    if (s.k == 1) return launch_rn_bwd<TX, TO, V, 1>(p, s, st);
    if (s.k == 2) return launch_rn_bwd<TX, TO, V, 2>(p, s, st);
    return launch_rn_bwd<TX, TO, V, 4>(p, s, st);
  }
  if (s.k == 2) return launch_rn_bwd<TX, TO, 1, 2>(p, s, st);
  if (s.k == 4) return launch_rn_bwd<TX, TO, 1, 4>(p, s, st);
  return launch_rn_bwd<TX, TO, 1, 16>(p, s, st);
}

template int rn_bwd<float, float>(RnParams&, bool, cudaStream_t);
template int rn_bwd<bf16, bf16>(RnParams&, bool, cudaStream_t);
template int rn_bwd<f16, f16>(RnParams&, bool, cudaStream_t);
template int rn_bwd<float, bf16>(RnParams&, bool, cudaStream_t);
template int rn_bwd<float, f16>(RnParams&, bool, cudaStream_t);

}  // namespace kda
