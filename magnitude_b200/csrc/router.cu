// The router of an expert layer: every row's logits, the experts it picks and their weights.
//
// Sums are held in 64 bits: a row's experts then depend neither on the order of its sum nor on the rows beside it, and two logits
// that differ in the last place of fp32 are told apart the same way in every batch.  bf16 x fp32 and fp32 x fp32 products are exact
// in a double.
#include <algorithm>

#include "router.h"

namespace b200q {

namespace {

constexpr int kThreads = 256, kWarps = 8;

// D += A (16 x 8 fp64, row) * B (8 x 8, col)
__device__ __forceinline__ void mma_f64(double (&c)[4], double a0, double a1, double a2, double a3, double b0, double b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f64.f64.f64.f64 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+d"(c[0]), "+d"(c[1]), "+d"(c[2]), "+d"(c[3])
        : "d"(a0), "d"(a1), "d"(a2), "d"(a3), "d"(b0), "d"(b1));
}

// eight elements from k0 on; zeros beyond K
__device__ __forceinline__ void load8(const void *base, long long at, int k0, int K, bool bf16, bool vec, float (&v)[8]) {
    if (bf16) {
        const unsigned short *src = reinterpret_cast<const unsigned short *>(base) + at + k0;
        if (vec && k0 + 8 <= K) {
            const uint4 w = *reinterpret_cast<const uint4 *>(src);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(word_of(w, i) << 16);
                v[2 * i + 1] = __uint_as_float(word_of(w, i) & 0xFFFF0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k0 + i < K ? __uint_as_float((uint32_t)src[i] << 16) : 0.f;
        }
    } else {
        const float *src = reinterpret_cast<const float *>(base) + at + k0;
        if (vec && k0 + 8 <= K) {
            const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k0 + i < K ? src[i] : 0.f;
        }
    }
}

// A block owns RT x 16 rows and ET x 8 experts; its warps split K in turns of 32 and are added up in order.
template <int RT, int ET>
__global__ void __launch_bounds__(kThreads) router_logits_kernel(const __grid_constant__ RouterRun p) {
    __shared__ double part[kWarps][32][4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.y * 16 * RT, e0 = blockIdx.x * 8 * ET;
    pdl_launch_dependents();
    pdl_wait();
    double acc[RT][ET][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < ET; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[r][e][i] = 0.0;
    const int chunks = (p.K + 31) / 32;
    for (int c = warp; c < chunks; c += kWarps) {
        const int k0 = c * 32 + 8 * t;
        float w[ET][8];
#pragma unroll
        for (int e = 0; e < ET; ++e) load8(p.w, (long long)min(e0 + 8 * e + g, p.experts - 1) * p.w_ld, k0, (int)p.w_ld, p.w_is_bf16, true, w[e]);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float x[2][8];
#pragma unroll
            for (int h = 0; h < 2; ++h) load8(p.x, (long long)min(row0 + 16 * r + 8 * h + g, p.m - 1) * p.ldx, k0, p.K, p.x_is_bf16, p.x_vec, x[h]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < ET; ++e) mma_f64(acc[r][e], x[0][2 * j], x[1][2 * j], x[0][2 * j + 1], x[1][2 * j + 1], w[e][2 * j], w[e][2 * j + 1]);
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < ET; ++e) {
#pragma unroll
            for (int i = 0; i < 4; ++i) part[warp][lane][i] = acc[r][e][i];
            __syncthreads();
            if (threadIdx.x < 128) {
                const int l = threadIdx.x >> 2, i = threadIdx.x & 3;
                double s = 0.0;
                for (int v = 0; v < kWarps; ++v) s += part[v][l][i];
                const int row = row0 + 16 * r + (l >> 2) + 8 * (i >> 1), ex = e0 + 8 * e + 2 * (l & 3) + (i & 1);
                if (row < p.m && ex < p.experts) p.logits[(long long)row * p.experts + ex] = s + (p.logit_bias ? (double)p.logit_bias[ex] : 0.0);
            }
            __syncthreads();
        }
}

// One warp per row: expert e belongs to lane e % 32.
template <int PER> __global__ void __launch_bounds__(kThreads) router_choose_kernel(const __grid_constant__ RouterRun p) {
    const int row = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();
    if (row >= p.m) return;
    constexpr double kMax = 1.7976931348623157e308;
    double score[PER], key[PER];             // key: what is compared; taken ones and those beyond the last expert fall below all others
    double top = -kMax;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = 32 * i + lane;
        double l = e < p.experts ? p.logits[(long long)row * p.experts + e] : -kMax;
        l = isnan(l) ? -kMax : fmin(fmax(l, -kMax), kMax);
        top = fmax(top, l);
        score[i] = p.sigmoid ? 1.0 / (1.0 + exp(-l)) : l;
        double k = score[i] + (p.select_bias && e < p.experts ? (double)p.select_bias[e] : 0.0);
        key[i] = isnan(k) ? -kMax : fmin(fmax(k, -kMax), kMax);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    float all = 0.f;                          // softmax over all experts
    if (!p.sigmoid && !p.normalise) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (32 * i + lane < p.experts) s += exp(score[i] - top);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
        all = (float)s;
    }
    unsigned left = 0;                        // experts of this lane that are still to have
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (32 * i + lane < p.experts) left |= 1u << i;
    float mine = 0.f, sum = 0.f;              // lane j keeps choice j's weight
    for (int j = 0; j < p.top_k; ++j) {
        double best = -kMax, s = 0.0;
        int at = 0x7FFFFFFF;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (((left >> i) & 1) && (at == 0x7FFFFFFF || key[i] > best)) best = key[i], at = 32 * i + lane, s = score[i];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const double ob = __shfl_xor_sync(0xFFFFFFFFu, best, d), os = __shfl_xor_sync(0xFFFFFFFFu, s, d);
            const int oa = __shfl_xor_sync(0xFFFFFFFFu, at, d);
            if (oa != 0x7FFFFFFF && (at == 0x7FFFFFFF || ob > best || (ob == best && oa < at))) best = ob, at = oa, s = os;
        }
        if ((at & 31) == lane) left &= ~(1u << (at >> 5));
        const float v = p.sigmoid ? (float)s : (float)exp(s - top);
        sum += v;
        if (lane == j) {
            mine = v;
            p.ids[row * p.ld_ids + j] = at;
        }
    }
    if (lane < p.top_k) {
        const float by = p.normalise ? sum : p.sigmoid ? 1.f : all;
        p.weights[row * p.ld_weights + lane] = by > 0.f ? mine / by * p.scale : 0.f;
    }
}

template <typename Kernel> cudaError_t launch(Kernel kern, const RouterRun &p, dim3 grid, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

cudaError_t router_run(const RouterRun &r, int sm_count, cudaStream_t st) {
    const unsigned rows16 = (unsigned)((r.m + 15) / 16), e8 = (unsigned)((r.experts + 7) / 8);
    // two row tiles and four expert tiles a block where that still gives every SM one: each operand is then converted once for several products
    cudaError_t e = (rows16 + 1) / 2 * ((e8 + 3) / 4) >= (unsigned)sm_count / 2 ? launch(router_logits_kernel<2, 4>, r, dim3((e8 + 3) / 4, (rows16 + 1) / 2), st)
                                                                              : launch(router_logits_kernel<1, 1>, r, dim3(e8, rows16), st);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)((r.m + kWarps - 1) / kWarps));
    if (r.experts <= 128) return launch(router_choose_kernel<4>, r, grid, st);
    if (r.experts <= 256) return launch(router_choose_kernel<8>, r, grid, st);
    return launch(router_choose_kernel<32>, r, grid, st);
}

}  // namespace b200q
