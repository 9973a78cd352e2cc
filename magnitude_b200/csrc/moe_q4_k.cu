// Expert layers: Q4_K weights.
#include "moe_kernel.cuh"

MOE_INSTANTIATE(q4_k, QT_Q4_K)
