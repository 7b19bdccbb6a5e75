#include "norm_fwd.cuh"

template int kda::rn_fwd<float, float>(kda::RnParams&, bool, cudaStream_t);
