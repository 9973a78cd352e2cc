// An expert layer for one row: two launches, no lists and no images in memory.
//
// What bounds a single row is not its bytes (2 us of weights in 128 experts of 2048 x 768) but the chain of launches, each of which
// waits for all of the one before.  So gate_up converts the row itself, and down converts the activations of all choices itself, while the weights
// are on their way: every warp keeps a ring of records of its own, filled by its own copies, and no warp waits for another before the sums over K
// are joined.  Two blocks an SM; down's blocks start as gate_up's leave and fetch their first records (which experts it will be is
// known by then) before the last activations are there.
// Measured, 128 experts of 2048 x 768, 8 of them, Q4_K / Q6_K: 13.1 us, 6.7 + 6.4 (with one block an SM for gate_up 16.4; by lists, images and
// cut units 23.7).
#pragma once

#include "moe_kernel.cuh"

namespace b200q {
namespace {

constexpr int kOneThreads = 32 * kMoeWarps;

template <int QT> constexpr int moe_one_depth() { return QT == QT_Q8_0 ? 2 : 3; }
template <int QT> constexpr int moe_one_ring() { return kMoeWarps * moe_one_depth<QT>() * moe_rec_bytes(QT); }

// elements k .. k + 7 of a row (past L1: the block may be older than they are)
__device__ __forceinline__ void moe_one_load(const void *x, int k, int K, bool bf16, bool vec, float (&v)[8]) {
    if (k >= K) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
    } else if (bf16) {
        const unsigned short *src = reinterpret_cast<const unsigned short *>(x) + k;
        if (vec) {
            const uint4 w = __ldcg(reinterpret_cast<const uint4 *>(src));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(word_of(w, i) << 16);
                v[2 * i + 1] = __uint_as_float(word_of(w, i) & 0xFFFF0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float((uint32_t)__ldcg(src + i) << 16);
        }
    } else {
        const float *src = reinterpret_cast<const float *>(x) + k;
        if (vec) {
            const float4 a = __ldcg(reinterpret_cast<const float4 *>(src)), b = __ldcg(reinterpret_cast<const float4 *>(src) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __ldcg(src + i);
        }
    }
}

template <int P> struct MoeOneShared {
    uint64_t bars[kMoeWarps][3];
    float part[2][kMoeWarps][16];        // the warps' sums over their records, of this unit and the one before
    __align__(16) uint8_t zero[256 * P];
    int fail;
};
// the sums of a tile's 16 rows over the warps, in the order of K: lane r < 16 of the calling warp has row r's
template <int P> __device__ __forceinline__ float moe_one_sum(const MoeOneShared<P> &s, int i, int lane) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kMoeWarps; ++w) sum += s.part[i & 1][w][lane & 15];
    return sum;
}
// gate, up and the activation function.  A unit is a choice and a tile of eight gate and eight up rows; the warps split K record by record,
// and convert of the row what they multiply.
template <int QT, int P> __global__ void __launch_bounds__(kOneThreads, 2) moe_one_gate_up_kernel(const __grid_constant__ MoeOneGateUp p) {
    constexpr int D = moe_one_depth<QT>(), REC = moe_rec_bytes(QT), IMG = moe_image_bytes(P);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ MoeOneShared<P> sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2;
    const MoeWeights &w = p.weights;
    uint8_t *images = smem + moe_one_ring<QT>(), *records = smem + warp * D * REC;
    WarpRing<D> ring;
    ring.init(sh.bars[warp], records, REC, lane);
    for (int i = tid; i < 64 * P; i += kOneThreads) reinterpret_cast<uint32_t *>(sh.zero)[i] = 0u;
    if (tid == 0) sh.fail = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();             // (from here on: down may read the choices)
    const int id = lane < p.choice.top_k ? __ldcg(p.choice.ids + lane) : -1;
    const int units = p.choice.top_k * w.tiles;
    auto expert_of = [&](int u) { return __shfl_sync(0xFFFFFFFFu, id, u / w.tiles); };
    // the record that is fetched next: unit fu, record fr
    int fu = blockIdx.x, fr = warp;
    const uint8_t *from = nullptr;
    int step = 0;                        // bytes from record to record of the tile
    auto seek = [&]() {                  // from fu on, the first unit that has an expert
        for (; fu < units; fu += gridDim.x) {
            const int e = expert_of(fu);
            if ((unsigned)e < (unsigned)p.choice.experts) {
                const int tile = fu % w.tiles;
                from = w.w + e * w.expert_bytes + moe_record_at(tile, 0, w.tiles, w.nrec) * REC;
                step = min(kMoeWarps, w.tiles - tile / kMoeWarps * kMoeWarps) * REC;
                break;
            }
        }
    };
    auto fetch = [&]() {
        if (fr >= w.nrec || fu >= units) return;
        ring.fill(from + (long long)fr * step, REC, lane);
        fr += kMoeWarps;
        if (fr >= w.nrec && warp < w.nrec) fr = warp, fu += gridDim.x, seek();
    };
    seek();
    for (int i = 0; i < D; ++i) fetch();
    for (int r = warp; r < w.nrec; r += kMoeWarps) {
        float v[8];
        moe_one_load(p.x.x, r * 256 + lane * 8, p.x.K, p.x.x_is_bf16, p.x.vec_ok, v);
        moe_image<P>(v, lane, images + r * IMG);
    }
    __syncwarp();
    const MoeColumns<1> col = moe_columns<P, 1>(1, lane);
    int i = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int e = expert_of(u);
        if ((unsigned)e >= (unsigned)p.choice.experts) continue;
        const int slot = u / w.tiles, tile = u - slot * w.tiles;
        float acc[1][2] = {{0.f, 0.f}};
        for (int r = warp; r < w.nrec; r += kMoeWarps) {
            ring.wait(&sh.fail, p.status);
            if (!ring.ok) break;
            MoeRecord<QT, P>::template run<MoeMode<1, 8 / (P == 2 ? 2 : 4)>>(records + ring.stage * REC, lane, images + r * IMG, sh.zero, col, acc);
            __syncwarp();
            fetch();
            ring.next();
        }
        moe_join<P, 1>(col, acc);
        if (col.row == 0) {
            sh.part[i & 1][warp][g] = acc[0][0];
            sh.part[i & 1][warp][g + 8] = acc[0][1];
        }
        __syncthreads();
        if (warp == i % kMoeWarps) {
            const float sum = moe_one_sum(sh, i, lane), up = __shfl_down_sync(0xFFFFFFFFu, sum, 8);
            const int f = tile * 8 + lane;
            if (lane < 8 && f < p.act.ff) p.h[(long long)slot * p.act.ff + f] = moe_activate(p.act, (long long)e * p.act.ff + f, sum, up);
        }
        ++i;
    }
    ring_leave(&sh.fail);
}

// down and the weighted sum over the choices.  A unit is a tile of 16 rows, its records are those of all choices one after the other; a warp takes
// an equal run of them.
template <int QT, int P> __global__ void __launch_bounds__(kOneThreads, 2) moe_one_down_kernel(const __grid_constant__ MoeOneDown p) {
    constexpr int D = moe_one_depth<QT>(), REC = moe_rec_bytes(QT), IMG = moe_image_bytes(P);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ MoeOneShared<P> sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2;
    const MoeWeights &w = p.weights;
    const MoeOutput &o = p.out;
    const int ff = p.ff, all = p.choice.top_k * w.nrec, j0 = all * warp / kMoeWarps, j1 = all * (warp + 1) / kMoeWarps;
    uint8_t *images = smem + moe_one_ring<QT>(), *records = smem + warp * D * REC;
    WarpRing<D> ring;
    ring.init(sh.bars[warp], records, REC, lane);
    for (int i = tid; i < 64 * P; i += kOneThreads) reinterpret_cast<uint32_t *>(sh.zero)[i] = 0u;
    if (tid == 0) sh.fail = 0;
    __syncthreads();
    pdl_launch_dependents();
    // gate_up's blocks, all of which had their choices when this block started, let it start: the choices are there, the activations not yet
    const int id = lane < p.choice.top_k ? __ldcg(p.choice.ids + lane) : -1;
    const float weight = lane < p.choice.top_k ? __ldcg(p.choice.weights + lane) : 0.f;
    auto chosen = [&](int c) { return (unsigned)__shfl_sync(0xFFFFFFFFu, id, c) < (unsigned)p.choice.experts; };
    // fetched next: tile ft, record fj of the run (choice fc, its record fk)
    int ft = blockIdx.x, fj = j0;
    auto fetch = [&]() {                 // one record, past those of choices without an expert
        while (ft < w.tiles && j0 < j1) {
            const int c = fj / w.nrec, r = fj - c * w.nrec, t = ft, e = __shfl_sync(0xFFFFFFFFu, id, c);
            if (++fj == j1) fj = j0, ft += gridDim.x;
            if ((unsigned)e < (unsigned)p.choice.experts) {
                ring.fill(w.w + e * w.expert_bytes + moe_record_at(t, r, w.tiles, w.nrec) * REC, REC, lane);
                return;
            }
        }
    };
    for (int i = 0; i < D; ++i) fetch();
    pdl_wait();
    for (int j = j0; j < j1; ++j) {
        const int c = j / w.nrec, r = j - c * w.nrec;
        if (!chosen(c)) continue;
        float v[8];
        moe_one_load(p.h + (long long)c * ff, r * 256 + lane * 8, ff, false, ff % 4 == 0, v);
        moe_image<P>(v, lane, images + j * IMG);
    }
    __syncwarp();
    const MoeColumns<1> col = moe_columns<P, 1>(1, lane);
    int i = 0;
    for (int tile = blockIdx.x; tile < w.tiles; tile += gridDim.x, ++i) {
        float total[1][2] = {{0.f, 0.f}};
        for (int j = j0; j < j1;) {
            const int c = j / w.nrec, next = min(j1, (c + 1) * w.nrec);
            if (!chosen(c)) {
                j = next;
                continue;
            }
            float acc[1][2] = {{0.f, 0.f}};
            for (; j < next; ++j) {
                ring.wait(&sh.fail, p.status);
                if (!ring.ok) break;
                MoeRecord<QT, P>::template run<MoeMode<1, 8 / (P == 2 ? 2 : 4)>>(records + ring.stage * REC, lane, images + j * IMG, sh.zero, col, acc);
                __syncwarp();
                fetch();
                ring.next();
            }
            j = next;
            const float by = __shfl_sync(0xFFFFFFFFu, weight, c);
            total[0][0] = fmaf(by, acc[0][0], total[0][0]);
            total[0][1] = fmaf(by, acc[0][1], total[0][1]);
        }
        moe_join<P, 1>(col, total);
        if (col.row == 0) {
            sh.part[i & 1][warp][g] = total[0][0];
            sh.part[i & 1][warp][g + 8] = total[0][1];
        }
        __syncthreads();
        if (warp == i % kMoeWarps) {
            float sum = moe_one_sum(sh, i, lane);
            const int n = tile * 16 + lane;
            const bool stores = lane < 16 && n < o.n;
            if (o.bias)
                for (int c = 0; c < p.choice.top_k; ++c) {
                    const int e = __shfl_sync(0xFFFFFFFFu, id, c);
                    const float by = __shfl_sync(0xFFFFFFFFu, weight, c);
                    if (stores && (unsigned)e < (unsigned)p.choice.experts) sum = fmaf(by, o.bias[(long long)e * o.n + n], sum);
                }
            if (stores && *(volatile int *)&sh.fail == 0) moe_store(o, 0, n, sum);
        }
    }
    ring_leave(&sh.fail);
}

}  // namespace
}  // namespace b200q

// bytes of shared memory beside which a row's images of `records` records lie
#define MOE_ONE_INSTANTIATE(NAME, QT)                                                                                              \
    namespace b200q {                                                                                                             \
    size_t moe_one_smem_##NAME(int planes, int records) { return (size_t)moe_one_ring<QT>() + (size_t)records * moe_image_bytes(planes); } \
    cudaError_t moe_one_gate_up_##NAME(const MoeOneGateUp &p, int planes, int grid, cudaStream_t st) {                              \
        const size_t smem = moe_one_smem_##NAME(planes, p.weights.nrec);                                                            \
        return planes == 2 ? moe_launch(moe_one_gate_up_kernel<QT, 2>, p, grid, smem, st, kOneThreads) : moe_launch(moe_one_gate_up_kernel<QT, 4>, p, grid, smem, st, kOneThreads); \
    }                                                                                                                             \
    cudaError_t moe_one_down_##NAME(const MoeOneDown &p, int planes, int grid, cudaStream_t st) {                                   \
        const size_t smem = moe_one_smem_##NAME(planes, p.choice.top_k * p.weights.nrec);                                           \
        return planes == 2 ? moe_launch(moe_one_down_kernel<QT, 2>, p, grid, smem, st, kOneThreads) : moe_launch(moe_one_down_kernel<QT, 4>, p, grid, smem, st, kOneThreads); \
    }                                                                                                                             \
    }
