// Expert layers: Q6_K weights.
#include "moe_kernel.cuh"

MOE_INSTANTIATE(q6_k, QT_Q6_K)
