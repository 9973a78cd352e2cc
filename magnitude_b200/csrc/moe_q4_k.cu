// Expert layers: Q4_K weights.
#include "moe_one.cuh"

MOE_INSTANTIATE(q4_k, QT_Q4_K)
MOE_ONE_INSTANTIATE(q4_k, QT_Q4_K)
