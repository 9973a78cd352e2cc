// Host side of the expert layer, and the launches around its products: the weights' re-layout, the lists of rows by expert, the
// activations' images.
#include <algorithm>

#include "moe_types.h"
#include "kernels.h"

namespace b200q {

namespace {

// ---- weights ---------------------------------------------------------------------------------------

// level k of a row of GGUF blocks, as the bits that the type packs it in
__device__ __forceinline__ int moe_level(int qt, const uint8_t *row, int64_t k) {
    const int i = (int)(k & 255);
    switch (qt) {
    case QT_Q4_K: return (row[(k >> 8) * 144 + 16 + 32 * (i >> 6) + (i & 31)] >> (i & 32 ? 4 : 0)) & 15;
    case QT_Q5_K: {
        const uint8_t *b = row + (k >> 8) * 176;
        return ((b[48 + 32 * (i >> 6) + (i & 31)] >> (i & 32 ? 4 : 0)) & 15) | ((b[16 + (i & 31)] >> (i >> 5)) & 1) << 4;
    }
    case QT_Q6_K: {
        const uint8_t *b = row + (k >> 8) * 210;
        const int half = i >> 7, run = (i >> 5) & 3, l = i & 31;
        return ((b[64 * half + 32 * (run & 1) + l] >> (run & 2 ? 4 : 0)) & 15) | ((b[128 + 32 * half + l] >> (2 * run)) & 3) << 4;
    }
    case QT_Q8_0: return row[(k >> 5) * 34 + 2 + (i & 31)];
    case QT_Q4_0: return (row[(k >> 5) * 18 + 2 + (i & 15)] >> (i & 16 ? 4 : 0)) & 15;
    default: return (row[(k >> 5) * 17 + 1 + (i & 15)] >> (i & 16 ? 4 : 0)) & 15;
    }
}

struct MoeRepack {
    int qt;
    const uint8_t *src[2];           // gate and up, or down twice
    uint8_t *dst;
    long long src_expert, dst_expert;   // bytes of an expert
    long long row_bytes;
    int rows, K, tiles, nrec;
    int paired;
};

// one warp per record
__global__ void __launch_bounds__(256) moe_repack_kernel(const MoeRepack p, long long records) {
    const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (id >= records) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rec = (int)(id % p.nrec), tile = (int)(id / p.nrec % p.tiles);
    const long long expert = id / p.nrec / p.tiles;
    uint8_t *out = p.dst + expert * p.dst_expert + ((long long)tile * p.nrec + rec) * moe_rec_bytes(p.qt);
    // row i of the tile, or null beyond the matrix
    auto row_of = [&](int i) -> const uint8_t * {
        const int r = p.paired ? tile * 8 + (i & 7) : tile * 16 + i;
        return r < p.rows ? p.src[p.paired && i >= 8] + expert * p.src_expert + r * p.row_bytes : nullptr;
    };
    const uint8_t *rows[2] = {row_of(g), row_of(g + 8)};
    // level of weight j of block b in word w of the lane's row; zero weights beyond K
    auto level = [&](int r, int b, int w, int j) -> int {
        const int64_t k = (int64_t)rec * 256 + 32 * b + 16 * w + 4 * t + j;
        const int none = p.qt == QT_Q6_K ? 32 : p.qt == QT_Q4_0 ? 8 : 0;
        return rows[r] && k < p.K ? moe_level(p.qt, rows[r], k) : none;
    };
    auto word4 = [&](auto byte) -> uint32_t { return (uint32_t)byte(0) | (uint32_t)byte(1) << 8 | (uint32_t)byte(2) << 16 | (uint32_t)byte(3) << 24; };
    uint4 *vec = reinterpret_cast<uint4 *>(out);
    auto put = [&](int v, auto word) { vec[v * 32 + lane] = make_uint4(word(0, 0), word(0, 1), word(1, 0), word(1, 1)); };      // word(row, w)
    if (p.qt == QT_Q8_0) {
        for (int b = 0; b < 8; ++b) put(b, [&](int r, int w) { return word4([&](int j) { return level(r, b, w, j); }); });
    } else if (p.qt == QT_MXFP4) {
        for (int v = 0; v < 4; ++v)
            put(v, [&](int r, int blk) {
                uint32_t x = 0;
                for (int i = 0; i < 8; ++i) x |= (uint32_t)level(r, 2 * v + blk, i >> 2, i & 3) << (4 * i);
                return x;
            });
    } else if (p.qt == QT_Q6_K) {
        for (int h = 0; h < 2; ++h)
            for (int n = 0; n < 3; ++n)
                put(3 * h + n, [&](int r, int e) {
                    const int q = 2 * n + e, tri = 2 * h + q / 3, part = q % 3;        // word `part` of triple tri
                    return word4([&](int j) {
                        // signed byte 4 (level - 32): the upper six bits; the fourth word's six bits lie two by two below the three
                        const int own = (level(r, 2 * tri + part / 2, part & 1, j) ^ 32) << 2;
                        const int fourth = level(r, 2 * tri + 1, 1, j) ^ 32;
                        return own | ((fourth >> (4 - 2 * part)) & 3);
                    });
                });
    } else {
        for (int v = 0; v < 4; ++v)
            put(v, [&](int r, int w) { return word4([&](int j) { return (level(r, 2 * v, w, j) & 15) | (level(r, 2 * v + 1, w, j) & 15) << 4; }); });
        if (p.qt == QT_Q5_K)
            put(4, [&](int r, int w) {
                return word4([&](int j) {
                    int bits = 0;
                    for (int b = 0; b < 8; ++b) bits |= (level(r, b, w, j) >> 4) << b;
                    return bits;
                });
            });
    }
    // the rows' scales: lane i < 16 writes row i's
    if (lane >= 16) return;
    const uint8_t *row = row_of(lane);
    uint8_t head[18] = {0};
    int bytes = 16, at = 2048;
    if (row) {
        if (p.qt == QT_Q4_K || p.qt == QT_Q5_K) {
            for (int i = 0; i < 16; ++i) head[i] = row[rec * (p.qt == QT_Q4_K ? 144 : 176) + i];
        } else if (p.qt == QT_Q6_K) {
            for (int i = 0; i < 18; ++i) head[i] = row[rec * 210 + 192 + i];
        } else {
            const int size = gguf_block_bytes(p.qt), each = p.qt == QT_MXFP4 ? 1 : 2;
            for (int b = 0; b < 8; ++b)
                if (rec * 8 + b < p.K / 32)
                    for (int i = 0; i < each; ++i) head[each * b + i] = row[(long long)(rec * 8 + b) * size + i];
        }
    }
    if (p.qt == QT_Q5_K) at = 2560;
    if (p.qt == QT_Q6_K) at = 3072;
    if (p.qt == QT_Q8_0) at = 4096;
    if (p.qt == QT_MXFP4) bytes = 8;
    for (int i = 0; i < bytes; ++i) out[at + bytes * lane + i] = head[i];
    if (p.qt == QT_Q6_K) out[3328 + 2 * lane] = head[16], out[3328 + 2 * lane + 1] = head[17];
}

// ---- activations -> images --------------------------------------------------------------------------

// 256 elements, eight a lane, into their image
template <int P> __device__ __forceinline__ void moe_image(const float (&v)[8], int lane, uint8_t *img) {
    uint32_t top = 0;                    // largest magnitude as bits: orders infinities and NaN above every number
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    const bool bad = top > __float_as_uint(3.0e38f);
    float mul, unit;
    if (P == 2) {
        // 16 bits: steps of largest / 32512 (127 * 256, so that the upper byte stays signed); below kTiny a fixed step
        constexpr float kMax = 32512.f, kTiny = 9.6e-35f;
        const float amax = fmaxf(__uint_as_float(top), kTiny);
        mul = kMax / amax;
        unit = amax * (1.f / kMax);
    } else {
        // a power of two that brings the largest to 2^29 .. 2^30: fp32 elements down to 2^-6 of it enter whole
        const int e = max((int)(top >> 23) - 127, -97);
        mul = __uint_as_float((uint32_t)(29 - e + 127) << 23);
        unit = __uint_as_float((uint32_t)(e - 29 + 127) << 23);
    }
    const int b = lane >> 2, l4 = lane & 3;
    uint32_t word[P][2];
#pragma unroll
    for (int p = 0; p < P; ++p) word[p][0] = word[p][1] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        int q = bad ? 0 : __float2int_rn(v[i] * mul);
#pragma unroll
        for (int p = P - 1; p >= 0; --p) {         // lowest plane last in the row
            const int d = p == 0 ? q : (int)(int8_t)q;
            word[p][i >> 2] |= (uint32_t)(d & 0xFF) << (8 * (i & 3));
            q = (q - d) >> 8;
        }
    }
    uint8_t *at = img + (b >> 1) * (64 * P) + (b & 1) * 8 + (l4 >> 1) * 4 + 32 * (l4 & 1);
#pragma unroll
    for (int p = 0; p < P; ++p) {
        *reinterpret_cast<uint32_t *>(at + 64 * p) = word[p][0];
        *reinterpret_cast<uint32_t *>(at + 64 * p + 16) = word[p][1];
        int s = dp4a_ss(word[p][0], 0x01010101u, dp4a_ss(word[p][1], 0x01010101u, 0));
        s += __shfl_xor_sync(0xFFFFFFFFu, s, 1);
        s += __shfl_xor_sync(0xFFFFFFFFu, s, 2);
        if (l4 == 0) {
            const int a = (s + 32) >> 6;
            uint8_t *sums = img + 256 * P + 16 * p + 8 * (b >> 2) + (b & 3);
            sums[0] = (uint8_t)a;
            sums[4] = (uint8_t)(s - 64 * a);
        }
    }
    if (lane < P / 2) {
        const float u = bad ? __int_as_float(0x7FC00000) : unit * (P == 4 && lane == 0 ? 65536.f : 1.f);
        reinterpret_cast<float *>(img + 272 * P)[lane] = u;
    }
}

struct MoeRows {
    const void *x;
    long long ldx;
    int x_is_bf16, vec_ok;
    int rows, K, nrec;
    uint8_t *img;
    unsigned img_stride;
    const int *ids;                      // rows are slots: those whose expert is none are left out
    long long ld_ids;
    int top_k, experts;
};

template <int P> __device__ __forceinline__ void moe_make_image(const MoeRows &p, long long task, int lane) {
    const int row = (int)(task / p.nrec), rec = (int)(task - (long long)row * p.nrec);
    if (p.ids && (unsigned)p.ids[row / p.top_k * p.ld_ids + row % p.top_k] >= (unsigned)p.experts) return;
    const int k0 = rec * 256 + lane * 8;
    float v[8];
    if (k0 >= p.K) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
    } else if (p.x_is_bf16) {
        const __nv_bfloat16 *src = reinterpret_cast<const __nv_bfloat16 *>(p.x) + row * p.ldx + k0;
        if (p.vec_ok) {
            const uint4 w = *reinterpret_cast<const uint4 *>(src);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(word_of(w, i) << 16);
                v[2 * i + 1] = __uint_as_float(word_of(w, i) & 0xFFFF0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(src[i]);
        }
    } else {
        const float *src = reinterpret_cast<const float *>(p.x) + row * p.ldx + k0;
        if (p.vec_ok) {
            const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = src[i];
        }
    }
    moe_image<P>(v, lane, p.img + (size_t)row * p.img_stride + (size_t)rec * moe_image_bytes(P));
}

// ---- lists -------------------------------------------------------------------------------------------

struct MoePrep {
    MoeRows rows;
    const int *ids;
    long long ld_ids;
    int m, top_k, experts, group;        // group: rows of a group at most
    MoeLists lists;
};

// Slots by expert, in ascending order within one, so that the same choice gives the same groups every time.  The block's threads own
// consecutive experts and read all ids.
__device__ void moe_make_lists(const MoePrep &p) {
    __shared__ int ids[kMoeMaxSlots];
    __shared__ int sums[8];
    const int slots = p.m * p.top_k, tid = threadIdx.x, lane = tid & 31;
    for (int s = tid; s < slots; s += 256) ids[s] = p.ids[s / p.top_k * p.ld_ids + s % p.top_k];
    __syncthreads();
    const int per = (p.experts + 255) / 256, e0 = tid * per;
    int count[kMoeMaxExperts / 256];
    int mine = 0;                        // groups
#pragma unroll
    for (int i = 0; i < kMoeMaxExperts / 256; ++i) {
        count[i] = 0;
        if (i < per && e0 + i < p.experts) {
            for (int s = 0; s < slots; ++s) count[i] += ids[s] == e0 + i;
            mine += (count[i] + p.group - 1) / p.group;
        }
    }
    int run = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, run, d);
        if (lane >= d) run += y;
    }
    if (lane == 31) sums[tid >> 5] = run;
    __syncthreads();
    int at = run - mine;
    for (int w = 0; w < (tid >> 5); ++w) at += sums[w];
    if (tid == 255) *p.lists.ngroups = at + mine;
#pragma unroll
    for (int i = 0; i < kMoeMaxExperts / 256; ++i) {
        if (i >= per || count[i] == 0) continue;
        int n = 0;
        for (int s = 0; s < slots; ++s)
            if (ids[s] == e0 + i) {
                MoeGroup &g = p.lists.groups[at];
                g.slot[n++] = s;
                --count[i];
                if (n == p.group || count[i] == 0) {
                    g.expert = e0 + i;
                    g.n = n;
                    n = 0;
                    ++at;
                }
            }
    }
}

// block 0: the lists; the others: the rows' images, one warp per record
template <int P> __global__ void __launch_bounds__(256) moe_prep_kernel(const __grid_constant__ MoePrep p) {
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0) {
        moe_make_lists(p);
        return;
    }
    const long long tasks = (long long)p.rows.rows * p.rows.nrec;
    for (long long task = (long long)(blockIdx.x - 1) * 8 + (threadIdx.x >> 5); task < tasks; task += (long long)(gridDim.x - 1) * 8)
        moe_make_image<P>(p.rows, task, threadIdx.x & 31);
}

template <int P> __global__ void __launch_bounds__(256) moe_image_kernel(const __grid_constant__ MoeRows p) {
    pdl_launch_dependents();
    pdl_wait();
    const long long tasks = (long long)p.rows * p.nrec;
    for (long long task = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); task < tasks; task += (long long)gridDim.x * 8)
        moe_make_image<P>(p, task, threadIdx.x & 31);
}

// y[m] = sum over the row's choices, in their order
struct MoeCombine {
    const float *z;
    long long ld_z;
    const int *ids;
    long long ld_ids;
    const float *weights;
    long long ld_weights;
    const float *bias;                   // [expert][n] or null
    void *y;
    long long ldy;
    int y_is_bf16, accumulate, n, m, top_k, experts;
};
__global__ void __launch_bounds__(256) moe_combine_kernel(const __grid_constant__ MoeCombine p) {
    pdl_launch_dependents();
    pdl_wait();
    const int n = blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
    if (n >= p.n) return;
    float sum = 0.f;
    for (int j = 0; j < p.top_k; ++j) {
        const int e = p.ids[m * p.ld_ids + j];
        if ((unsigned)e >= (unsigned)p.experts) continue;
        float v = p.z[(long long)(m * p.top_k + j) * p.ld_z + n];
        if (p.bias) v += p.bias[(long long)e * p.n + n];
        sum = fmaf(p.weights[m * p.ld_weights + j], v, sum);
    }
    const long long at = m * p.ldy + n;
    if (p.y_is_bf16) {
        __nv_bfloat16 *y = reinterpret_cast<__nv_bfloat16 *>(p.y) + at;
        *y = __float2bfloat16_rn(p.accumulate ? __bfloat162float(*y) + sum : sum);
    } else {
        float *y = reinterpret_cast<float *>(p.y) + at;
        *y = p.accumulate ? *y + sum : sum;
    }
}

template <typename Kernel, typename Params> cudaError_t launch(Kernel kern, const Params &p, dim3 grid, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void *args[] = {const_cast<Params *>(&p)};
    return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void *>(kern), args);
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

cudaError_t gate_up_launch(int qt, const MoeGateUp &p, const MoeConfig &c, int grid, cudaStream_t st) {
    switch (qt) {
    case QT_Q4_K: return moe_gate_up_q4_k(p, c, grid, st);
    case QT_Q5_K: return moe_gate_up_q5_k(p, c, grid, st);
    case QT_Q6_K: return moe_gate_up_q6_k(p, c, grid, st);
    case QT_Q8_0: return moe_gate_up_q8_0(p, c, grid, st);
    case QT_Q4_0: return moe_gate_up_q4_0(p, c, grid, st);
    default: return moe_gate_up_mxfp4(p, c, grid, st);
    }
}
cudaError_t down_launch(int qt, const MoeDown &p, const MoeConfig &c, int grid, cudaStream_t st) {
    switch (qt) {
    case QT_Q4_K: return moe_down_q4_k(p, c, grid, st);
    case QT_Q5_K: return moe_down_q5_k(p, c, grid, st);
    case QT_Q6_K: return moe_down_q6_k(p, c, grid, st);
    case QT_Q8_0: return moe_down_q8_0(p, c, grid, st);
    case QT_Q4_0: return moe_down_q4_0(p, c, grid, st);
    default: return moe_down_mxfp4(p, c, grid, st);
    }
}

}  // namespace

size_t moe_matrix_bytes(int qt, int64_t experts, int64_t rows, int64_t K, bool paired) {
    return (size_t)experts * ceil_div(rows, paired ? 8 : 16) * ceil_div(K, SB) * moe_rec_bytes(qt);
}

cudaError_t moe_repack(int qt, const uint8_t *src0, const uint8_t *src1, uint8_t *dst, int64_t experts, int64_t rows, int64_t K, cudaStream_t st) {
    MoeRepack p{};
    p.qt = qt;
    p.paired = src1 != nullptr;
    p.src[0] = src0;
    p.src[1] = src1 ? src1 : src0;
    p.dst = dst;
    p.row_bytes = K / gguf_block_elems(qt) * gguf_block_bytes(qt);
    p.src_expert = rows * p.row_bytes;
    p.rows = (int)rows;
    p.K = (int)K;
    p.tiles = (int)ceil_div(rows, p.paired ? 8 : 16);
    p.nrec = (int)ceil_div(K, SB);
    p.dst_expert = (long long)p.tiles * p.nrec * moe_rec_bytes(qt);
    const long long records = experts * p.tiles * p.nrec;
    moe_repack_kernel<<<(unsigned)ceil_div(records, 8), 256, 0, st>>>(p, records);
    return cudaGetLastError();
}

// Bytes of the workspace of a layer of up to max_rows rows, and where its parts lie.
size_t moe_workspace(const MoeShapeInfo &s, MoeBuffers *out, uint8_t *base) {
    const int64_t slots = s.max_rows * s.top_k;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return base ? base + here : nullptr;
    };
    MoeBuffers b{};
    b.lists.ngroups = reinterpret_cast<int *>(take(sizeof(int)));
    b.lists.groups = reinterpret_cast<MoeGroup *>(take(sizeof(MoeGroup) * (size_t)slots));
    b.h = reinterpret_cast<float *>(take(sizeof(float) * (size_t)(slots * s.n_ff)));
    b.x_img = take((size_t)s.max_rows * ceil_div(s.n_embd, SB) * moe_image_bytes(4));
    b.h_img = take((size_t)slots * ceil_div(s.n_ff, SB) * moe_image_bytes(4));
    b.z = reinterpret_cast<float *>(take((size_t)slots * ceil_div(s.n_embd, 16) * 16 * sizeof(float)));
    if (out) *out = b;
    return at;
}

cudaError_t moe_run(const MoeRun &r, cudaStream_t st, int *launches) {
    const MoeShapeInfo &s = r.shape;
    const int slots = r.m * (int)s.top_k;
    // 31-bit activations for fp32 results, 16 bits where the result is rounded to bf16
    MoeConfig c{};
    c.planes = r.y_is_bf16 ? 2 : 4;
    c.column_tiles = r.m * c.planes <= 8 ? 1 : 4;
    const int x_rec = (int)ceil_div(s.n_embd, SB), h_rec = (int)ceil_div(s.n_ff, SB);

    MoePrep pr{};
    pr.rows.x = r.x;
    pr.rows.ldx = r.ldx;
    pr.rows.x_is_bf16 = r.x_is_bf16;
    pr.rows.vec_ok = (reinterpret_cast<uintptr_t>(r.x) & 15) == 0 && (r.ldx * (r.x_is_bf16 ? 2 : 4)) % 16 == 0;
    pr.rows.rows = r.m;
    pr.rows.K = (int)s.n_embd;
    pr.rows.nrec = x_rec;
    pr.rows.img = r.buf.x_img;
    pr.rows.img_stride = (unsigned)(x_rec * moe_image_bytes(c.planes));
    pr.ids = r.ids;
    pr.ld_ids = r.ld_ids;
    pr.m = r.m;
    pr.top_k = (int)s.top_k;
    pr.experts = (int)s.n_experts;
    pr.group = moe_group_rows(c.planes, c.column_tiles);
    pr.lists = r.buf.lists;
    const int prep_grid = 1 + (int)std::min<long long>(ceil_div((long long)r.m * x_rec, 8), 4 * s.sm_count);
    cudaError_t e = c.planes == 2 ? launch(moe_prep_kernel<2>, pr, prep_grid, st) : launch(moe_prep_kernel<4>, pr, prep_grid, st);
    if (e != cudaSuccess) return e;

    const int used = (int)std::min<long long>(slots, s.n_experts);      // experts that may have been chosen
    // Records of a tile are shared by as many warps as it takes to give every warp of the chip work
    auto product = [&](const uint8_t *w, int qt, int tiles, int nrec, const uint8_t *img, unsigned stride, int per_row) {
        MoeProduct p{};
        p.w = w;
        p.tiles = tiles;
        p.nrec = nrec;
        p.expert_bytes = (long long)tiles * nrec * moe_rec_bytes(qt);
        p.lists = r.buf.lists;
        p.img = img;
        p.img_stride = stride;
        p.slots_per_row = per_row;
        p.status = r.status;
        p.split = 1;
        while (p.split < moe_max_split(qt, c.planes, c.column_tiles) && 2 * p.split <= nrec && (long long)used * tiles * p.split < 2ll * kMoeWarps * s.sm_count) p.split *= 2;
        return p;
    };
    auto grid_of = [&](const MoeProduct &p) {
        return (int)std::min<long long>(2 * s.sm_count, (long long)slots * ceil_div(p.tiles, kMoeWarps / p.split));
    };
    MoeGateUp gu{};
    gu.product = product(r.gate_up, r.gate_up_type, (int)ceil_div(s.n_ff, 8), x_rec, r.buf.x_img, pr.rows.img_stride, (int)s.top_k);
    gu.h = r.buf.h;
    gu.ff = (int)s.n_ff;
    gu.activation = r.activation;
    gu.alpha = r.alpha;
    gu.limit = r.limit;
    gu.gate_bias = r.gate_bias;
    gu.up_bias = r.up_bias;
    if ((e = gate_up_launch(r.gate_up_type, gu, c, grid_of(gu.product), st)) != cudaSuccess) return e;

    MoeRows hr{};
    hr.x = r.buf.h;
    hr.ldx = s.n_ff;
    hr.vec_ok = s.n_ff % 4 == 0;
    hr.rows = slots;
    hr.K = (int)s.n_ff;
    hr.nrec = h_rec;
    hr.img = r.buf.h_img;
    hr.img_stride = (unsigned)(h_rec * moe_image_bytes(c.planes));
    hr.ids = r.ids;
    hr.ld_ids = r.ld_ids;
    hr.top_k = (int)s.top_k;
    hr.experts = (int)s.n_experts;
    const int h_grid = (int)std::min<long long>(ceil_div((long long)slots * h_rec, 8), 4 * s.sm_count);
    e = c.planes == 2 ? launch(moe_image_kernel<2>, hr, h_grid, st) : launch(moe_image_kernel<4>, hr, h_grid, st);
    if (e != cudaSuccess) return e;

    MoeDown d{};
    d.product = product(r.down, r.down_type, (int)ceil_div(s.n_embd, 16), h_rec, r.buf.h_img, hr.img_stride, 1);
    d.z = r.buf.z;
    d.ld_z = ceil_div(s.n_embd, 16) * 16;
    if ((e = down_launch(r.down_type, d, c, grid_of(d.product), st)) != cudaSuccess) return e;

    MoeCombine cb{};
    cb.z = d.z;
    cb.ld_z = d.ld_z;
    cb.ids = r.ids;
    cb.ld_ids = r.ld_ids;
    cb.weights = r.weights;
    cb.ld_weights = r.ld_weights;
    cb.bias = r.down_bias;
    cb.y = r.y;
    cb.ldy = r.ldy;
    cb.y_is_bf16 = r.y_is_bf16;
    cb.accumulate = r.accumulate;
    cb.n = (int)s.n_embd;
    cb.m = r.m;
    cb.top_k = (int)s.top_k;
    cb.experts = (int)s.n_experts;
    if ((e = launch(moe_combine_kernel, cb, dim3((unsigned)ceil_div(s.n_embd, 256), (unsigned)r.m), st)) != cudaSuccess) return e;
    *launches = 5;
    return cudaSuccess;
}

cudaError_t moe_set_wait_limit_ns(unsigned long long ns) {
    cudaError_t e;
    for (auto set : {moe_wait_limit_q4_k, moe_wait_limit_q5_k, moe_wait_limit_q6_k, moe_wait_limit_q8_0, moe_wait_limit_q4_0, moe_wait_limit_mxfp4})
        if ((e = set(ns)) != cudaSuccess) return e;
    return cudaSuccess;
}

}  // namespace b200q
