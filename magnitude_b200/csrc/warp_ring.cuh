// A ring of pieces in shared memory that belongs to one warp: the warp asks for its pieces by bulk copies, ahead of their use, and no warp
// waits for another one's.
#pragma once

#include "common.cuh"

namespace b200q {
namespace {

// One bounded wait by all lanes; on expiry (or when another warp already gave up) the warp leaves
__device__ __forceinline__ bool ring_wait(uint32_t bar, uint32_t parity, volatile int *fail, int *status) {
    if (mbar_try_wait_hint(bar, parity, 32)) return true;
    if (*fail) return false;
    if (mbar_wait_bounded_fast(bar, parity)) return true;
    atomicMax(status, DEV_ERR_PIPE_TIMEOUT);
    *fail = 1;
    return false;
}
// Called by all threads at the end: after a failure copies may still be on their way, and get time to land (far above a copy's latency)
// before the block's shared memory is released.
__device__ __forceinline__ void ring_leave(volatile int *fail) {
    __syncthreads();
    if (*fail) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 100000) {
        }
    }
}

template <int D> struct WarpRing {
    uint32_t bars, at, piece;        // D barriers, D pieces
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    bool ok = true;
    __device__ __forceinline__ void init(uint64_t *bar, const uint8_t *smem, uint32_t piece_bytes, int lane) {
        bars = smem_u32(bar);
        at = smem_u32(smem);
        piece = piece_bytes;
        if (lane == 0) {
            for (int i = 0; i < D; ++i) mbar_init(bars + 8 * i, 1);
            mbar_fence_init();
            fence_proxy_async();
        }
        __syncwarp();
    }
    // the next piece into the stage after the last one filled, which is free: its readers have met since (__syncwarp).  (No proxy fence: reads
    // that are over need none before a copy, and a fence would wait for the global loads that the warp has on their way, too.)
    __device__ __forceinline__ void fill(const void *src, uint32_t bytes, int lane) {
        if (lane == 0) {
            mbar_expect_tx(bars + 8 * filled, bytes);
            bulk_g2s(at + filled * piece, src, bytes, bars + 8 * filled);
        }
        if (++filled == D) filled = 0;
    }
    __device__ __forceinline__ void wait(volatile int *fail, int *status) { ok = ok && __all_sync(0xFFFFFFFFu, ring_wait(bars + 8 * stage, phase, fail, status)); }
    __device__ __forceinline__ void next() {
        if (++stage == D) stage = 0, phase ^= 1;
    }
};

}  // namespace
}  // namespace b200q
