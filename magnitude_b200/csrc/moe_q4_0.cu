// Expert layers: Q4_0 weights.
#include "moe_kernel.cuh"

MOE_INSTANTIATE(q4_0, QT_Q4_0)
