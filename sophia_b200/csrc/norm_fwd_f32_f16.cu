#include "norm_fwd.cuh"

template int kda::rn_fwd<float, kda::f16>(kda::RnParams&, bool, cudaStream_t);
