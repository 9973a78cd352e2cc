// Expert layers: Q8_0 weights.
#include "moe_one.cuh"

MOE_INSTANTIATE(q8_0, QT_Q8_0)
MOE_ONE_INSTANTIATE(q8_0, QT_Q8_0)
