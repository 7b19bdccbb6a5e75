#include "norm_bwd.cuh"

template int kda::rn_bwd<float, float>(kda::RnParams&, bool, cudaStream_t);
