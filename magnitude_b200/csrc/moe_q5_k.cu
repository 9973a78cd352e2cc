// Expert layers: Q5_K weights.
#include "moe_kernel.cuh"

MOE_INSTANTIATE(q5_k, QT_Q5_K)
