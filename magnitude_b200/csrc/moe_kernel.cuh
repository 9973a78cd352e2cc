// The products of an expert layer: every group of rows that chose an expert against that expert's weights.
//
// A warp multiplies 16 weight rows by the 8 / P activation rows of a column tile, 256 weights a step, with
// mma.m16n8k32 on bytes: weight levels as they are (one or two logic operations per four weights), activations in P byte
// planes that are columns of their own.  Every MMA stays inside one block of 32 weights (Q6_K: m16n8k16, one of
// 16); its integer sums are multiplied by the block's integer scale and added up as integers over the record (Q4_K, Q5_K,
// Q6_K), or scaled in fp32 (types with an fp16 or power-of-two scale per block), so nothing is multiplied per weight.  The
// minima of Q4_K and Q5_K are two more MMAs with the sums of the activations' blocks.
// A block takes one group and the records of eight tile rows a step (its warps one each), through a ring of stages that hold the
// weights and the group's activations; the warps share the activations.
#pragma once

#include "kernels.h"
#include "moe_types.h"

namespace b200q {
namespace {

// D = A (16 x 32 bytes) * B (32 x 8 signed bytes)
template <bool SIGNED> __device__ __forceinline__ void moe_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (SIGNED)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
// D = A (16 x 16 signed bytes) * B (16 x 8)
__device__ __forceinline__ void moe_mma16(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "r"(0));
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ int byte_u(uint32_t w, int i) { return (w >> (8 * i)) & 0xFF; }
__device__ __forceinline__ int byte_s(uint32_t w, int i) { return (int)(int8_t)(w >> (8 * i)); }

// where a lane finds its column of a column tile in the group's images: byte offsets
template <int NT> struct MoeColumns {
    int b[NT];               // the bytes of column g (lane >> 2), its t's share
    int s[NT];               // the scale of columns 2 t, 2 t + 1
    int live;                // column tiles that hold rows
};

__device__ __forceinline__ uint4 moe_lds(const uint8_t *p) { return *reinterpret_cast<const uint4 *>(p); }
// the lane's B words of block pair j: x, y of block 2 j, z, w of block 2 j + 1
template <int P> __device__ __forceinline__ uint4 moe_b(const uint8_t *img, int j) { return moe_lds(img + j * (64 * P)); }

// One record: acc[nt][0], [1] += rows g, g + 8 against the column tile's columns 2 t, 2 t + 1 (one plane pair).
// rec: the record, img: the group's images of this record, both in shared memory
template <int QT, int P, int NT> struct MoeRecord;

// Q4_K, Q5_K
template <int QT, int P, int NT> struct MoeRecordK {
    static __device__ __forceinline__ void run(const uint8_t *rec, int lane, const uint8_t *img, const MoeColumns<NT> &col, float (&acc)[NT][2]) {
        const int g = lane >> 2, t = lane & 3;
        constexpr int kHead = QT == QT_Q5_K ? 2560 : 2048;
        uint4 hd[2], f;
        hd[0] = moe_lds(rec + kHead + 16 * g);
        hd[1] = moe_lds(rec + kHead + 16 * g + 128);
        if (QT == QT_Q5_K) f = moe_lds(rec + 2048 + 16 * lane);
        uint32_t sc[2][2], am[2];            // scales of blocks 0 .. 3, 4 .. 7; minima of blocks 4 t .. as an A word (t < 2)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sc[i][0] = hd[i].y & 0x3F3F3F3Fu;
            sc[i][1] = (hd[i].w & 0x0F0F0F0Fu) | ((hd[i].y >> 2) & 0x30303030u);
            const uint32_t m1 = ((hd[i].w >> 4) & 0x0F0F0F0Fu) | ((hd[i].z >> 2) & 0x30303030u);
            am[i] = t == 0 ? hd[i].z & 0x3F3F3F3Fu : t == 1 ? m1 : 0u;
        }
        int even[NT][4], odd[NT][4];         // Q4_K: high nibbles enter as 16 x level and are added up apart
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) even[nt][x] = odd[nt][x] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint4 q = moe_lds(rec + 512 * j + 16 * lane);
            uint32_t lo[4], hi[4];           // [row g: words 0, 1][row g + 8: words 0, 1]
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t v = word_of(q, i);
                if (QT == QT_Q4_K) {
                    lo[i] = v & 0x0F0F0F0Fu;
                    hi[i] = v & 0xF0F0F0F0u;
                } else {
                    const uint32_t b = word_of(f, i);
                    const uint32_t b0 = 2 * j < 4 ? b << (4 - 2 * j) : b >> (2 * j - 4), b1 = 2 * j + 1 < 4 ? b << (3 - 2 * j) : b >> (2 * j - 3);
                    lo[i] = (v & 0x0F0F0F0Fu) | (b0 & 0x10101010u);
                    hi[i] = ((v >> 4) & 0x0F0F0F0Fu) | (b1 & 0x10101010u);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (nt > 0 && nt >= col.live) break;
                const uint4 b = moe_b<P>(img + col.b[nt], j);
                int c[4];
                moe_mma<false>(c, lo[0], lo[2], lo[1], lo[3], b.x, b.y);
#pragma unroll
                for (int x = 0; x < 4; ++x) even[nt][x] += c[x] * byte_u(sc[x >> 1][j >> 1], 2 * (j & 1));
                moe_mma<false>(c, hi[0], hi[2], hi[1], hi[3], b.z, b.w);
#pragma unroll
                for (int x = 0; x < 4; ++x) odd[nt][x] += c[x] * byte_u(sc[x >> 1][j >> 1], 2 * (j & 1) + 1);
            }
        }
        const float scale = QT == QT_Q4_K ? 0.0625f : 1.f;
        float d[2], dmin[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            d[i] = half_bits_to_float(hd[i].x) * scale;
            dmin[i] = half_bits_to_float(hd[i].x >> 16);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt > 0 && nt >= col.live) break;
            // block sums 64 a + b: lanes t < 2 bring a and b of blocks 4 t .. 4 t + 3, the others' A words are zero
            const uint2 bs = *reinterpret_cast<const uint2 *>(img + col.b[nt] + 256 * P - 48 * (g % P) - 16 * t + 8 * (t & 1));
            int ma[4], mb[4];
            moe_mma<false>(ma, am[0], am[1], 0u, 0u, bs.x, 0u);
            moe_mma<false>(mb, am[0], am[1], 0u, 0u, bs.y, 0u);
            const float s = *reinterpret_cast<const float *>(img + col.s[nt]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int v0 = QT == QT_Q4_K ? 16 * even[nt][2 * i] + odd[nt][2 * i] : even[nt][2 * i] + odd[nt][2 * i];
                const int v1 = QT == QT_Q4_K ? 16 * even[nt][2 * i + 1] + odd[nt][2 * i + 1] : even[nt][2 * i + 1] + odd[nt][2 * i + 1];
                const float v = fmaf(256.f, (float)v0, (float)v1);
                const float m = fmaf(256.f, (float)(64 * ma[2 * i] + mb[2 * i]), (float)(64 * ma[2 * i + 1] + mb[2 * i + 1]));
                acc[nt][i] = fmaf(s, fmaf(d[i], v, -dmin[i] * m), acc[nt][i]);
            }
        }
    }
};
template <int P, int NT> struct MoeRecord<QT_Q4_K, P, NT> : MoeRecordK<QT_Q4_K, P, NT> {};
template <int P, int NT> struct MoeRecord<QT_Q5_K, P, NT> : MoeRecordK<QT_Q5_K, P, NT> {};

template <int P, int NT> struct MoeRecord<QT_Q6_K, P, NT> {
    static __device__ __forceinline__ void run(const uint8_t *rec, int lane, const uint8_t *img, const MoeColumns<NT> &col, float (&acc)[NT][2]) {
        const int g = lane >> 2;
        const uint4 s0 = moe_lds(rec + 3072 + 16 * g), s1 = moe_lds(rec + 3072 + 16 * g + 128);
        const float d[2] = {half_bits_to_float(*reinterpret_cast<const uint16_t *>(rec + 3328 + 2 * g)) * 0.25f, half_bits_to_float(*reinterpret_cast<const uint16_t *>(rec + 3328 + 2 * g + 16)) * 0.25f};
        int sum[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) sum[nt][x] = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // six words a row: triples 2 h, 2 h + 1
            uint32_t w[2][6];
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                const uint4 v = moe_lds(rec + 512 * (3 * h + n) + 16 * lane);
                w[0][2 * n] = v.x, w[0][2 * n + 1] = v.y, w[1][2 * n] = v.z, w[1][2 * n + 1] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {            // blocks 2 j, 2 j + 1 with j = 2 h + i
                const int j = 2 * h + i;
                uint32_t a[2][4];                     // four 16-weight sub-blocks
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t x = w[r][3 * i], y = w[r][3 * i + 1], z = w[r][3 * i + 2];
                    a[r][0] = x & 0xFCFCFCFCu;
                    a[r][1] = y & 0xFCFCFCFCu;
                    a[r][2] = z & 0xFCFCFCFCu;
                    a[r][3] = ((x << 6) & 0xC0C0C0C0u) | ((y << 4) & 0x30303030u) | ((z << 2) & 0x0C0C0C0Cu);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (nt > 0 && nt >= col.live) break;
                    const uint4 b = moe_b<P>(img + col.b[nt], j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        int c[4];
                        moe_mma16(c, a[0][e], a[1][e], word_of(b, e));
#pragma unroll
                        for (int x = 0; x < 4; ++x) sum[nt][x] += c[x] * byte_s(word_of(x < 2 ? s0 : s1, j), e);
                    }
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt > 0 && nt >= col.live) break;
            const float s = *reinterpret_cast<const float *>(img + col.s[nt]);
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[nt][i] = fmaf(s, d[i] * fmaf(256.f, (float)sum[nt][2 * i], (float)sum[nt][2 * i + 1]), acc[nt][i]);
        }
    }
};

// types with one scale per 32 weights
template <int QT, int P, int NT> struct MoeRecordBlock {
    static __device__ __forceinline__ void run(const uint8_t *rec, int lane, const uint8_t *img, const MoeColumns<NT> &col, float (&acc)[NT][2]) {
        const int g = lane >> 2;
        uint4 hd[2];                                  // eight fp16 d (MXFP4: eight scale bytes)
        if (QT == QT_MXFP4) {
            const uint2 e0 = *reinterpret_cast<const uint2 *>(rec + 2048 + 8 * g), e1 = *reinterpret_cast<const uint2 *>(rec + 2048 + 8 * g + 64);
            hd[0] = make_uint4(e0.x, e0.y, 0, 0), hd[1] = make_uint4(e1.x, e1.y, 0, 0);
        } else {
            constexpr int kHead = QT == QT_Q8_0 ? 4096 : 2048;
            hd[0] = moe_lds(rec + kHead + 16 * g), hd[1] = moe_lds(rec + kHead + 16 * g + 128);
        }
        float e[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) e[nt][0] = e[nt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t a[2][4];                         // blocks 2 j, 2 j + 1: [row g: words 0, 1][row g + 8: words 0, 1]
            if (QT == QT_Q8_0) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint4 v = moe_lds(rec + 512 * (2 * j + b) + 16 * lane);
                    a[b][0] = v.x, a[b][1] = v.y, a[b][2] = v.z, a[b][3] = v.w;
                }
            } else {
                const uint4 v = moe_lds(rec + 512 * j + 16 * lane);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t q = word_of(v, i);
                    if (QT == QT_Q4_0) {              // 16 (level - 8) as signed bytes
                        a[0][i] = ((q << 4) & 0xF0F0F0F0u) ^ 0x80808080u;
                        a[1][i] = (q & 0xF0F0F0F0u) ^ 0x80808080u;
                    } else {                          // twice the value: 2 (64 + v) - 128
                        const uint32_t lo = mxfp4_bytes(q), hi = mxfp4_bytes(q >> 16);
                        a[i & 1][(i & 2)] = (lo + lo) ^ 0x80808080u;
                        a[i & 1][(i & 2) + 1] = (hi + hi) ^ 0x80808080u;
                    }
                }
            }
            float d[2][2];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int k = 2 * j + b;
                    if (QT == QT_MXFP4) d[r][b] = __uint_as_float(e8m0_half_bits(byte_u(k < 4 ? hd[r].x : hd[r].y, k & 3)));
                    else d[r][b] = half_bits_to_float(word_of(hd[r], j) >> (16 * b));
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (nt > 0 && nt >= col.live) break;
                const uint4 b = moe_b<P>(img + col.b[nt], j);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    int c[4];
                    moe_mma<true>(c, a[k][0], a[k][2], a[k][1], a[k][3], k ? b.z : b.x, k ? b.w : b.y);
                    e[nt][0] = fmaf(d[0][k], (float)(256 * c[0] + c[1]), e[nt][0]);
                    e[nt][1] = fmaf(d[1][k], (float)(256 * c[2] + c[3]), e[nt][1]);
                }
            }
        }
        constexpr float scale = QT == QT_Q8_0 ? 1.f : QT == QT_Q4_0 ? 0.0625f : 0.5f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt > 0 && nt >= col.live) break;
            const float s = *reinterpret_cast<const float *>(img + col.s[nt]) * scale;
            acc[nt][0] = fmaf(s, e[nt][0], acc[nt][0]);
            acc[nt][1] = fmaf(s, e[nt][1], acc[nt][1]);
        }
    }
};
template <int P, int NT> struct MoeRecord<QT_Q8_0, P, NT> : MoeRecordBlock<QT_Q8_0, P, NT> {};
template <int P, int NT> struct MoeRecord<QT_Q4_0, P, NT> : MoeRecordBlock<QT_Q4_0, P, NT> {};
template <int P, int NT> struct MoeRecord<QT_MXFP4, P, NT> : MoeRecordBlock<QT_MXFP4, P, NT> {};

// The lane's columns of a group of n rows: rows beyond the last repeat it (their sums are not stored)
template <int P, int NT> __device__ __forceinline__ MoeColumns<NT> moe_columns(int n, int lane) {
    constexpr int IMG = moe_image_bytes(P);
    const int g = lane >> 2, t = lane & 3;
    MoeColumns<NT> c;
    c.live = (n * P + 7) / 8;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        c.b[nt] = min(nt * (8 / P) + g / P, n - 1) * IMG + (g % P) * 64 + t * 16;
        c.s[nt] = min(nt * (8 / P) + 2 * t / P, n - 1) * IMG + P * 272 + 4 * ((2 * t % P) / 2);
    }
    return c;
}

// both plane pairs of a row (P = 4) are added up; every lane of a pair has the sum
template <int P, int NT> __device__ __forceinline__ void moe_join_planes(float (&acc)[NT][2]) {
    if (P == 4) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[nt][i] += __shfl_xor_sync(0xFFFFFFFFu, acc[nt][i], 1);
    }
}

// A product's part of one block: units (group, run of tiles) in turn, every unit's records a step at a time.  With `split` warps a tile
// (few tiles in all), a step takes as many records of 8 / split tiles, and the warps' sums are added up in order.
//   finish(unit's group, tile, acc): one warp per tile, its lanes hold the sums of rows g, g + 8 and columns 2 t, 2 t + 1
template <int QT, int P, int NT, typename Finish>
__device__ __forceinline__ void moe_product(const MoeProduct &p, uint8_t *smem, float (*part)[NT][2][32], Finish finish) {
    constexpr int REC = moe_rec_bytes(QT), D = moe_depth(QT, P, NT), IMG = moe_image_bytes(P), kGroup = moe_group_rows(P, NT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = p.split, per = kMoeWarps / split, ws = warp % split, wt = warp / split;     // the warp's record of a step and tile of a unit
    const int runs = (p.tiles + per - 1) / per, units = *p.lists.ngroups * runs, steps = (p.nrec + split - 1) / split;
    const int stage_bytes = moe_stage_bytes(QT, P, NT, split);

    // what is copied next
    int fu = blockIdx.x, fs = 0, put = 0;
    const uint8_t *w_src = nullptr;          // the warp's record
    uint32_t b_src[kMoeChunks];              // the thread's pieces of the images: offsets of the next step's
    int b_rec[kMoeChunks], b_dst[kMoeChunks];
    auto fetch = [&] {
        if (fu < units) {
            if (fs == 0) {
                const int gi = fu / runs, tile = (fu - gi * runs) * per + wt;
                const MoeGroup grp = p.lists.groups[gi];
                w_src = tile < p.tiles ? p.w + grp.expert * p.expert_bytes + ((long long)tile * p.nrec + ws) * REC : nullptr;
#pragma unroll
                for (int i = 0; i < kMoeChunks; ++i) {
                    const int piece = i * kMoeThreads + tid, row = piece / (IMG / 16), at = piece - row * (IMG / 16);     // row = (record of the step, row of the group)
                    const int s = row / grp.n, m = row - s * grp.n;
                    b_rec[i] = s < split ? s : 0x40000000;
                    b_dst[i] = (s * kGroup + m) * IMG + at * 16;
                    b_src[i] = s < split ? (uint32_t)(p.lists.sorted[grp.first + m] / p.slots_per_row) * p.img_stride + s * IMG + at * 16 : 0u;
                }
            }
            uint8_t *stage = smem + put * stage_bytes;
            if (w_src && fs * split + ws < p.nrec) {
                const uint32_t dst = smem_u32(stage + warp * REC) + 16 * lane;
#pragma unroll
                for (int i = 0; i < (REC / 16 + 31) / 32; ++i)
                    if ((REC / 16) % 32 == 0 || i * 32 + lane < REC / 16) cp_async_16(dst + 512 * i, w_src + 512 * i + 16 * lane);
            }
            if (w_src) w_src += split * REC;
            const uint32_t img = smem_u32(stage + kMoeWarps * REC);
#pragma unroll
            for (int i = 0; i < kMoeChunks; ++i) {
                if (b_rec[i] < p.nrec) cp_async_16(img + b_dst[i], p.img + b_src[i]);
                b_rec[i] += split;
                b_src[i] += split * IMG;
            }
            if (++fs == steps) fs = 0, fu += gridDim.x;
        }
        cp_async_commit();
        if (++put == D) put = 0;
    };
#pragma unroll
    for (int i = 0; i < D - 1; ++i) fetch();
    int get = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int gi = u / runs, tile = (u - gi * runs) * per + wt;
        const MoeGroup grp = p.lists.groups[gi];
        const MoeColumns<NT> col = moe_columns<P, NT>(grp.n, lane);
        float acc[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = 0.f;
        for (int s = 0; s < steps; ++s) {
            cp_async_wait<D - 2>();
            __syncthreads();                 // the stage is here, and the one before it has been read
            fetch();
            const uint8_t *stage = smem + get * stage_bytes;
            if (tile < p.tiles && s * split + ws < p.nrec)
                MoeRecord<QT, P, NT>::run(stage + warp * REC, lane, stage + kMoeWarps * REC + ws * kGroup * IMG, col, acc);
            if (++get == D) get = 0;
        }
        moe_join_planes<P, NT>(acc);
        if (split > 1) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) part[warp][nt][i][lane] = acc[nt][i];
            __syncthreads();                 // (the next unit's are written after at least one more)
            if (ws == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        for (int k = 1; k < split; ++k) acc[nt][i] += part[warp + k][nt][i][lane];
            }
        }
        if (ws == 0 && tile < p.tiles) finish(grp, tile, acc);
    }
    cp_async_wait<0>();
}

// ---- gate, up and the activation function --------------------------------------------------------
template <int QT, int P, int NT>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_gate_up_kernel(const __grid_constant__ MoeGateUp p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float part[kMoeWarps][NT][2][32];
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();
    moe_product<QT, P, NT>(p.product, smem, part, [&](const MoeGroup &grp, int tile, const float (&acc)[NT][2]) {
        const int f = tile * 8 + g;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * (8 / P) + 2 * t / P;
            if (f >= p.ff || r >= grp.n || (2 * t) % P) continue;
            float a = acc[nt][0], b = acc[nt][1];
            if (p.gate_bias) a += p.gate_bias[(long long)grp.expert * p.ff + f];
            if (p.up_bias) b += p.up_bias[(long long)grp.expert * p.ff + f];
            float h;
            if (p.activation == B200Q_MOE_SWIGLU_CLAMPED) {
                // (comparisons that keep NaN)
                a = a > p.limit ? p.limit : a;
                b = b > p.limit ? p.limit : b < -p.limit ? -p.limit : b;
                h = a / (1.f + expf(-p.alpha * a)) * (b + 1.f);
            } else {
                h = a / (1.f + expf(-a)) * b;
            }
            p.h[(long long)p.product.lists.sorted[grp.first + r] * p.ff + f] = h;
        }
    });
}

// ---- down ------------------------------------------------------------------------------------------
template <int QT, int P, int NT>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_down_kernel(const __grid_constant__ MoeDown p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float part[kMoeWarps][NT][2][32];
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();
    moe_product<QT, P, NT>(p.product, smem, part, [&](const MoeGroup &grp, int tile, const float (&acc)[NT][2]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * (8 / P) + 2 * t / P;
            if (r >= grp.n || (2 * t) % P) continue;
            float *z = p.z + (long long)p.product.lists.sorted[grp.first + r] * p.ld_z + tile * 16 + g;
            z[0] = acc[nt][0];
            z[8] = acc[nt][1];
        }
    });
}

template <typename Kernel, typename Params> cudaError_t moe_launch(Kernel kern, const Params &p, int grid, size_t smem, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kMoeThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void *args[] = {const_cast<Params *>(&p)};
    return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void *>(kern), args);
}

}  // namespace
}  // namespace b200q

// one source file per weight type (they compile side by side)
#define MOE_INSTANTIATE(NAME, QT)                                                                                                     \
    namespace b200q {                                                                                                                 \
    namespace {                                                                                                                       \
    size_t moe_smem(const MoeProduct &p, const MoeConfig &c) {                                                                          \
        return (size_t)moe_depth(QT, c.planes, c.column_tiles) * moe_stage_bytes(QT, c.planes, c.column_tiles, p.split);                   \
    }                                                                                                                                 \
    }                                                                                                                                 \
    cudaError_t moe_gate_up_##NAME(const MoeGateUp &p, const MoeConfig &c, int grid, cudaStream_t st) {                                 \
        const size_t smem = moe_smem(p.product, c);                                                                                     \
        if (c.planes == 2) return c.column_tiles == 1 ? moe_launch(moe_gate_up_kernel<QT, 2, 1>, p, grid, smem, st)                     \
                                                      : moe_launch(moe_gate_up_kernel<QT, 2, 4>, p, grid, smem, st);                    \
        return c.column_tiles == 1 ? moe_launch(moe_gate_up_kernel<QT, 4, 1>, p, grid, smem, st)                                        \
                                   : moe_launch(moe_gate_up_kernel<QT, 4, 4>, p, grid, smem, st);                                       \
    }                                                                                                                                 \
    cudaError_t moe_down_##NAME(const MoeDown &p, const MoeConfig &c, int grid, cudaStream_t st) {                                      \
        const size_t smem = moe_smem(p.product, c);                                                                                     \
        if (c.planes == 2) return c.column_tiles == 1 ? moe_launch(moe_down_kernel<QT, 2, 1>, p, grid, smem, st)                        \
                                                      : moe_launch(moe_down_kernel<QT, 2, 4>, p, grid, smem, st);                       \
        return c.column_tiles == 1 ? moe_launch(moe_down_kernel<QT, 4, 1>, p, grid, smem, st)                                           \
                                   : moe_launch(moe_down_kernel<QT, 4, 4>, p, grid, smem, st);                                          \
    }                                                                                                                                 \
    }
