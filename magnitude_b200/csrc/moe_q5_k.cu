// Expert layers: Q5_K weights.
#include "moe_one.cuh"

MOE_INSTANTIATE(q5_k, QT_Q5_K)
MOE_ONE_INSTANTIATE(q5_k, QT_Q5_K)
