// Expert layers: MXFP4 weights.
#include "moe_kernel.cuh"

MOE_INSTANTIATE(mxfp4, QT_MXFP4)
