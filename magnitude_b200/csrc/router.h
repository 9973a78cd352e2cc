// What the C ABI layer and the router's kernels (router.cu) share.
#pragma once

#include "common.cuh"

namespace b200q {

constexpr int kRouterMaxExperts = 1024, kRouterMaxTopK = 32, kRouterMaxRanges = 4;

struct RouterRun {
    const void *w;                   // [experts][w_ld], zeros beyond K
    long long w_ld;
    int w_is_bf16;
    const float *logit_bias, *select_bias;
    int experts, top_k, K;
    int sigmoid, normalise;
    float scale;
    const void *x;
    long long ldx;
    int x_is_bf16, x_vec;
    int m;
    int *ids;
    long long ld_ids;
    float *weights;
    long long ld_weights;
    double *logits;                  // [range of K][m][experts]
    int ranges;
    unsigned *count;                 // zero between launches
};

cudaError_t router_run(RouterRun r, int sm_count, cudaStream_t st);

}  // namespace b200q
