#include "norm_fwd.cuh"

template int kda::rn_fwd<kda::bf16, kda::bf16>(kda::RnParams&, bool, cudaStream_t);
