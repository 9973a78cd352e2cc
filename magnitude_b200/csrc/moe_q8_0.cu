// Expert layers: Q8_0 weights.
#include "moe_kernel.cuh"

MOE_INSTANTIATE(q8_0, QT_Q8_0)
