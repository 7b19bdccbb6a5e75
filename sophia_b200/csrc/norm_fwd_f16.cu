#include "norm_fwd.cuh"

template int kda::rn_fwd<kda::f16, kda::f16>(kda::RnParams&, bool, cudaStream_t);
