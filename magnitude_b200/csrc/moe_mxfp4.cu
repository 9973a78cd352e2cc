// Expert layers: MXFP4 weights.
#include "moe_one.cuh"

MOE_INSTANTIATE(mxfp4, QT_MXFP4)
MOE_ONE_INSTANTIATE(mxfp4, QT_MXFP4)
