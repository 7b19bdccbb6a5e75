#include "norm_bwd.cuh"

template int kda::rn_bwd<float, kda::f16>(kda::RnParams&, bool, cudaStream_t);
