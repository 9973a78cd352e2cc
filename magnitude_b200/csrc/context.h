// What the files of the C ABI layer share: the context, error reporting and argument helpers.
#pragma once

#include <stdarg.h>
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace b200q {

// What a call leaves in device memory between its launches.  Calls that share a set must be ordered by one stream.
struct Scratch {
    void *gemm_x = nullptr;           // fp16 copy of the activations
    size_t gemm_x_bytes = 0;
    void *dense_w = nullptr;          // fp16 weights of the two-launch GEMM, one panel at a time
    size_t dense_w_bytes = 0;
    float *gemm_part = nullptr;       // K-split partial products (allocated on first use)
    // small batches (2..48 rows): sums of tiles shared by several blocks, zero between launches
    uint8_t *sk_ws = nullptr;
    uint8_t *sk_img = nullptr;        // activation images
    size_t sk_img_bytes = 0;
    void free_all() {
        for (void *p : {gemm_x, dense_w, (void *)gemm_part, (void *)sk_ws, (void *)sk_img})
            if (p) cudaFree(p);
        *this = Scratch{};
    }
};

}  // namespace b200q

struct b200q_ctx {
    int device = 0;
    int sm_count = 0;
    size_t smem_optin = 0;
    size_t smem_sm = 0;
    int *status_dev = nullptr;
    char err[512] = {0};
    int last_route = B200Q_ROUTE_NONE;
    int last_launches = 0;
    bool poisoned = false;
    // host-buffer path
    cudaStream_t hstream = nullptr;
    void *hx_dev = nullptr;
    size_t hx_bytes = 0;
    void *hy_dev = nullptr;
    size_t hy_bytes = 0;
    b200q::Scratch scratch;                  // calls on the caller's stream
    b200q::Scratch hscratch;                 // host-buffer calls: the caller cannot order hstream after calls in flight on its own stream
    uint64_t tp_timeout_ms = 60000;   // host deadline of b200q_tp_init
    bool peer_stale = false;          // a peer exchange timed out: the ranks' call counters no longer agree
    bool peer_ipc = true;             // peer buffers were mapped through CUDA IPC (else given as pointers)
    int skinny_min_m = 3;             // smallest M that takes the skinny route (smaller batches: the streaming kernel)
    int mid_max_m = 48;               // largest M that runs on the small-batch kernels (17 and more rows)
    int gemm_bn = 0, gemm_debug = 0, gemm_pair = 0, gemm_ksplit = 1, gemm_dense = -1;
    // tunables (environment overrides for experiments)
    int gemv_grid = 0, gemv_smem = 0, gemv_pdl = 1, gemv_xprep = 1;
    float *adapter_t = nullptr;       // A x of large adapter calls (allocated with the first adapter set)
    // tensor parallel
    void *comm = nullptr;            // ncclComm_t
    int tp_rank = 0, tp_world = 1;
    // peer exchange (CUDA IPC): own buffer, every rank's buffer as mapped here
    uint8_t *peer_local = nullptr;
    uint8_t *peer_base[b200q::kPeerMaxWorld] = {nullptr};
    int peer_rank = -1, peer_world = 0;
};

namespace b200q {

b200q_status fail(b200q_ctx *ctx, b200q_status code, const char *fmt, ...);
b200q_status cuda_fail(b200q_ctx *ctx, cudaError_t e, const char *what);
// the context is usable and its device current
b200q_status check_ctx(b200q_ctx *ctx);

#define CU_TRY(ctx, expr)                                          \
    do {                                                           \
        cudaError_t e__ = (expr);                                  \
        if (e__ != cudaSuccess) return cuda_fail(ctx, e__, #expr); \
    } while (0)

inline bool known_type(int t) { return t == QT_MXFP4 || t == QT_Q4_0 || t == QT_Q8_0 || t == QT_Q4_K || t == QT_Q5_K || t == QT_Q6_K; }
inline bool act_type(int t) { return t == B200Q_TYPE_F32 || t == B200Q_TYPE_BF16; }
inline size_t act_size(int t) { return t == B200Q_TYPE_BF16 ? 2 : 4; }

}  // namespace b200q
