// Expert layers: Q6_K weights.
#include "moe_one.cuh"

MOE_INSTANTIATE(q6_k, QT_Q6_K)
MOE_ONE_INSTANTIATE(q6_k, QT_Q6_K)
