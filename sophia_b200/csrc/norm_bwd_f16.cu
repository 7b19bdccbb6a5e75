#include "norm_bwd.cuh"

template int kda::rn_bwd<kda::f16, kda::f16>(kda::RnParams&, bool, cudaStream_t);
