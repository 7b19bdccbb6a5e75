#include "norm_bwd.cuh"

template int kda::rn_bwd<kda::bf16, kda::bf16>(kda::RnParams&, bool, cudaStream_t);
