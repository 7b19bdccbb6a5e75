// The selective scan on bf16 activations.
#define SSM_SCAN_INSTANTIATE kda::bf16
#include "ssm_scan_launch.cuh"
