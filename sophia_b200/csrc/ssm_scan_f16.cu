// The selective scan on fp16 activations.
#define SSM_SCAN_INSTANTIATE kda::f16
#include "ssm_scan_launch.cuh"
