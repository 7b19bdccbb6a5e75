// The selective scan on fp32 activations.
#define SSM_SCAN_INSTANTIATE float
#include "ssm_scan_launch.cuh"
