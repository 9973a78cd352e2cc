// Expert layers: Q4_0 weights.
#include "moe_one.cuh"

MOE_INSTANTIATE(q4_0, QT_Q4_0)
MOE_ONE_INSTANTIATE(q4_0, QT_Q4_0)
