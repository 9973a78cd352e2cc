// The products of an expert layer: every group of rows that chose an expert against that expert's weights.
//
// A warp multiplies 16 weight rows by the 8 / P activation rows of a column tile, 256 weights a step, with
// mma.m16n8k32 on bytes: weight levels as they are (one or two logic operations per four weights), activations in P byte
// planes that are columns of their own.  Every MMA stays inside one block of 32 weights (Q6_K: m16n8k16, one of
// 16); its integer sums are multiplied by the block's integer scale and added up as integers over the record (Q4_K, Q5_K,
// Q6_K), or scaled in fp32 (types with an fp16 or power-of-two scale per block), so nothing is multiplied per weight.  The
// minima of Q4_K and Q5_K are two more MMAs with the sums of the activations' blocks.
// A block takes one group and the records of eight tile rows a step: a producer warp copies the weights and the group's activations
// into a ring of stages, eight warps multiply, one record each, and share the activations.
#pragma once

#include "kernels.h"
#include "moe_types.h"

namespace b200q {
namespace {

// D += A (16 x 32 bytes) * B (32 x 8 signed bytes); first: D = A * B
template <bool SIGNED> __device__ __forceinline__ void moe_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool first) {
    const int c0 = first ? 0 : d[0], c1 = first ? 0 : d[1], c2 = first ? 0 : d[2], c3 = first ? 0 : d[3];
    if (SIGNED)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}
// D += A (16 x 16 signed bytes) * B (16 x 8)
__device__ __forceinline__ void moe_mma16(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0, bool first) {
    const int c0 = first ? 0 : d[0], c1 = first ? 0 : d[1], c2 = first ? 0 : d[2], c3 = first ? 0 : d[3];
    asm("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %8, %9, %10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}

__device__ __forceinline__ int byte_u(uint32_t w, int i) { return __byte_perm(w, 0u, 0x4440 | i); }
// (the upper bit of a selector's digit repeats the byte's sign; __byte_perm leaves it out)
__device__ __forceinline__ int byte_s(uint32_t w, int i) {
    int v;
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(v) : "r"(w), "r"(0x1111 * i | 0x8880));
    return v;
}

// How a warp's columns are used.  NL column tiles hold 8 / P rows each.  A group of few rows needs only half or a quarter
// of one tile: then the columns also tell F blocks apart (column = class F, row, plane; class f holds blocks f, f + F, .. and zeros for the
// others), F MMAs add up into the same sums, and a lane has 1 / F of the scaling to do.
template <int NL_, int F_> struct MoeMode {
    static constexpr int NL = NL_, F = F_;
};

// where a lane finds its column in the group's images: byte offsets
template <int NT> struct MoeColumns {
    int b[NT];               // the bytes of column g (lane >> 2), its t's share
    int s[NT];               // the scale of columns 2 t, 2 t + 1
    int classes, class_b, class_s;      // F; the class of column g, of columns 2 t, 2 t + 1
    int row;                 // the row of columns 2 t, 2 t + 1 of the first tile; -1: the lane has nothing to store
};

__device__ __forceinline__ uint4 moe_lds(const uint8_t *p) { return *reinterpret_cast<const uint4 *>(p); }
// the lane's B words of block pair j: x, y of block 2 j, z, w of block 2 j + 1
template <int P> __device__ __forceinline__ uint4 moe_b(const uint8_t *img, int j) { return moe_lds(img + j * (64 * P)); }
template <int P> __device__ __forceinline__ uint2 moe_b_block(const uint8_t *img, int b) { return *reinterpret_cast<const uint2 *>(img + (b >> 1) * (64 * P) + 8 * (b & 1)); }

// One record: acc[nt][0], [1] += rows g, g + 8 against columns 2 t, 2 t + 1 (one plane pair) of column tile nt.
// rec: the record, img: the group's images of this record, zero: as many zeros, all in shared memory
template <int QT, int P> struct MoeRecord;

// Q4_K, Q5_K
template <int QT, int P> struct MoeRecordK {
    // A words of blocks 2 j (low nibbles) and 2 j + 1: [row g: words 0, 1][row g + 8: words 0, 1]
    static __device__ __forceinline__ void words(const uint8_t *rec, int lane, int j, const uint4 &f, uint32_t (&lo)[4], uint32_t (&hi)[4]) {
        const uint4 q = moe_lds(rec + 512 * j + 16 * lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = word_of(q, i);
            if (QT == QT_Q4_K) {
                lo[i] = v & 0x0F0F0F0Fu;
                hi[i] = v & 0xF0F0F0F0u;         // 16 x level
            } else {
                const uint32_t b = word_of(f, i);
                const uint32_t b0 = 2 * j < 4 ? b << (4 - 2 * j) : b >> (2 * j - 4), b1 = 2 * j + 1 < 4 ? b << (3 - 2 * j) : b >> (2 * j - 3);
                lo[i] = (v & 0x0F0F0F0Fu) | (b0 & 0x10101010u);
                hi[i] = ((v >> 4) & 0x0F0F0F0Fu) | (b1 & 0x10101010u);
            }
        }
    }
    template <typename Mode, int NT>
    static __device__ __forceinline__ void run(const uint8_t *rec, int lane, const uint8_t *img, const uint8_t *zero, const MoeColumns<NT> &col, float (&acc)[NT][2]) {
        constexpr int NL = Mode::NL, F = Mode::F;
        const int g = lane >> 2, t = lane & 3;
        constexpr int kHead = QT == QT_Q5_K ? 2560 : 2048;
        uint4 hd[2], f = make_uint4(0, 0, 0, 0);
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
        int sum[NL][4];
        float scale = 1.f;
        if (F == 1) {
            int odd[NL][4];                  // Q4_K: high nibbles are added up apart
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t lo[4], hi[4];
                words(rec, lane, j, f, lo, hi);
#pragma unroll
                for (int nt = 0; nt < NL; ++nt) {
                    const uint4 b = moe_b<P>(img + col.b[nt], j);
                    int c[4];
                    moe_mma<false>(c, lo[0], lo[2], lo[1], lo[3], b.x, b.y, true);
#pragma unroll
                    for (int x = 0; x < 4; ++x) sum[nt][x] = (j ? sum[nt][x] : 0) + c[x] * byte_u(sc[x >> 1][j >> 1], 2 * (j & 1));
                    moe_mma<false>(c, hi[0], hi[2], hi[1], hi[3], b.z, b.w, true);
                    int(&o)[4] = QT == QT_Q4_K ? odd[nt] : sum[nt];
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[x] = (j || QT != QT_Q4_K ? o[x] : 0) + c[x] * byte_u(sc[x >> 1][j >> 1], 2 * (j & 1) + 1);
                }
            }
            if (QT == QT_Q4_K) {
                scale = 0.0625f;
#pragma unroll
                for (int nt = 0; nt < NL; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) sum[nt][x] = 16 * sum[nt][x] + odd[nt][x];
            }
        } else {
            const uint8_t *bp[F];
#pragma unroll
            for (int r = 0; r < F; ++r) bp[r] = r == col.class_b ? img + col.b[0] : zero;
            int c[8 / F][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t lo[4], hi[4];
                words(rec, lane, j, f, lo, hi);
                const uint2 b0 = moe_b_block<P>(bp[2 * j % F], 2 * j), b1 = moe_b_block<P>(bp[(2 * j + 1) % F], 2 * j + 1);
                moe_mma<false>(c[2 * j / F], lo[0], lo[2], lo[1], lo[3], b0.x, b0.y, 2 * j % F == 0);
                moe_mma<false>(c[2 * j / F], hi[0], hi[2], hi[1], hi[3], b1.x, b1.y, false);
            }
            // the lane's blocks: F q + class
#pragma unroll
            for (int x = 0; x < 4; ++x) sum[0][x] = 0;
#pragma unroll
            for (int q = 0; q < 8 / F; ++q)
#pragma unroll
                for (int x = 0; x < 4; ++x) sum[0][x] += c[q][x] * byte_u(sc[x >> 1][q * F / 4], q * F % 4 + col.class_s);
            if (QT == QT_Q4_K && (col.class_s & 1)) scale = 0.0625f;
        }
        float d[2], dmin[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            d[i] = half_bits_to_float(hd[i].x) * scale;
            dmin[i] = F == 1 || col.class_s == 0 ? half_bits_to_float(hd[i].x >> 16) : 0.f;
        }
#pragma unroll
        for (int nt = 0; nt < NL; ++nt) {
            // block sums 64 a + b: lanes t < 2 bring a and b of blocks 4 t .. 4 t + 3, the others' A words are zero.  (class F's bytes begin
            // where the image does, so the plane follows from the offset)
            const int plane = F == 1 ? g % P : g % (8 / F) % P;
            const uint2 bs = *reinterpret_cast<const uint2 *>(img + col.b[nt] + 256 * P - 48 * plane - 16 * t + 8 * (t & 1));
            int ma[4], mb[4];
            moe_mma<false>(ma, am[0], am[1], 0u, 0u, bs.x, 0u, true);
            moe_mma<false>(mb, am[0], am[1], 0u, 0u, bs.y, 0u, true);
            const float s = *reinterpret_cast<const float *>(img + col.s[nt]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float v = fmaf(256.f, (float)sum[nt][2 * i], (float)sum[nt][2 * i + 1]);
                const float m = fmaf(256.f, (float)(64 * ma[2 * i] + mb[2 * i]), (float)(64 * ma[2 * i + 1] + mb[2 * i + 1]));
                acc[nt][i] = fmaf(s, fmaf(d[i], v, -dmin[i] * m), acc[nt][i]);
            }
        }
    }
};
template <int P> struct MoeRecord<QT_Q4_K, P> : MoeRecordK<QT_Q4_K, P> {};
template <int P> struct MoeRecord<QT_Q5_K, P> : MoeRecordK<QT_Q5_K, P> {};

template <int P> struct MoeRecord<QT_Q6_K, P> {
    template <typename Mode, int NT>
    static __device__ __forceinline__ void run(const uint8_t *rec, int lane, const uint8_t *img, const uint8_t *zero, const MoeColumns<NT> &col, float (&acc)[NT][2]) {
        constexpr int NL = Mode::NL, F = Mode::F;
        const int g = lane >> 2;
        const uint4 s0 = moe_lds(rec + 3072 + 16 * g), s1 = moe_lds(rec + 3072 + 16 * g + 128);
        const float d[2] = {half_bits_to_float(*reinterpret_cast<const uint16_t *>(rec + 3328 + 2 * g)) * 0.25f,
                            half_bits_to_float(*reinterpret_cast<const uint16_t *>(rec + 3328 + 2 * g + 16)) * 0.25f};
        const uint8_t *bp[F];
#pragma unroll
        for (int r = 0; r < F; ++r) bp[r] = F == 1 || r == col.class_b ? img + col.b[0] : zero;
        int sum[NL][4];
#pragma unroll
        for (int nt = 0; nt < NL; ++nt)
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
                if (F == 1) {
#pragma unroll
                    for (int nt = 0; nt < NL; ++nt) {
                        const uint4 b = moe_b<P>(img + col.b[nt], j);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            int c[4];
                            moe_mma16(c, a[0][e], a[1][e], word_of(b, e), true);
#pragma unroll
                            for (int x = 0; x < 4; ++x) sum[nt][x] += c[x] * byte_s(word_of(x < 2 ? s0 : s1, j), e);
                        }
                    }
                } else {
                    int c[4 / F][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        moe_mma16(c[e / F], a[0][e], a[1][e], *reinterpret_cast<const uint32_t *>(bp[e % F] + j * (64 * P) + 4 * e), e % F == 0);
#pragma unroll
                    for (int q = 0; q < 4 / F; ++q)
#pragma unroll
                        for (int x = 0; x < 4; ++x) sum[0][x] += c[q][x] * byte_s(word_of(x < 2 ? s0 : s1, j), q * F + col.class_s);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NL; ++nt) {
            const float s = *reinterpret_cast<const float *>(img + col.s[nt]);
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[nt][i] = fmaf(s, d[i] * fmaf(256.f, (float)sum[nt][2 * i], (float)sum[nt][2 * i + 1]), acc[nt][i]);
        }
    }
};

// types with one scale per 32 weights
template <int QT, int P> struct MoeRecordBlock {
    // scale of block k of a row from its header
    static __device__ __forceinline__ float scale_of(const uint4 &hd, int k) {
        if (QT == QT_MXFP4) return __uint_as_float(e8m0_half_bits(byte_u(k < 4 ? hd.x : hd.y, k & 3)));
        return half_bits_to_float((k < 4 ? (k < 2 ? hd.x : hd.y) : (k < 6 ? hd.z : hd.w)) >> (16 * (k & 1)));
    }
    template <typename Mode, int NT>
    static __device__ __forceinline__ void run(const uint8_t *rec, int lane, const uint8_t *img, const uint8_t *zero, const MoeColumns<NT> &col, float (&acc)[NT][2]) {
        constexpr int NL = Mode::NL, F = Mode::F;
        const int g = lane >> 2;
        uint4 hd[2];                                  // eight fp16 d (MXFP4: eight scale bytes)
        if (QT == QT_MXFP4) {
            const uint2 e0 = *reinterpret_cast<const uint2 *>(rec + 2048 + 8 * g), e1 = *reinterpret_cast<const uint2 *>(rec + 2048 + 8 * g + 64);
            hd[0] = make_uint4(e0.x, e0.y, 0, 0), hd[1] = make_uint4(e1.x, e1.y, 0, 0);
        } else {
            constexpr int kHead = QT == QT_Q8_0 ? 4096 : 2048;
            hd[0] = moe_lds(rec + kHead + 16 * g), hd[1] = moe_lds(rec + kHead + 16 * g + 128);
        }
        const uint8_t *bp[F];
#pragma unroll
        for (int r = 0; r < F; ++r) bp[r] = F == 1 || r == col.class_b ? img + col.b[0] : zero;
        float e[NL][2];
#pragma unroll
        for (int nt = 0; nt < NL; ++nt) e[nt][0] = e[nt][1] = 0.f;
        int cf[F == 1 ? 1 : 8 / F][4];
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
            if (F == 1) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float d0 = scale_of(hd[0], 2 * j + k), d1 = scale_of(hd[1], 2 * j + k);
#pragma unroll
                    for (int nt = 0; nt < NL; ++nt) {
                        const uint2 b = moe_b_block<P>(img + col.b[nt], 2 * j + k);
                        int c[4];
                        moe_mma<true>(c, a[k][0], a[k][2], a[k][1], a[k][3], b.x, b.y, true);
                        e[nt][0] = fmaf(d0, (float)(256 * c[0] + c[1]), e[nt][0]);
                        e[nt][1] = fmaf(d1, (float)(256 * c[2] + c[3]), e[nt][1]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int b = 2 * j + k;
                    const uint2 v = moe_b_block<P>(bp[b % F], b);
                    moe_mma<true>(cf[b / F], a[k][0], a[k][2], a[k][1], a[k][3], v.x, v.y, b % F == 0);
                }
            }
        }
        if (F > 1) {
#pragma unroll
            for (int q = 0; q < 8 / F; ++q) {
                const int b = q * F + col.class_s;
                e[0][0] = fmaf(scale_of(hd[0], b), (float)(256 * cf[q][0] + cf[q][1]), e[0][0]);
                e[0][1] = fmaf(scale_of(hd[1], b), (float)(256 * cf[q][2] + cf[q][3]), e[0][1]);
            }
        }
        constexpr float scale = QT == QT_Q8_0 ? 1.f : QT == QT_Q4_0 ? 0.0625f : 0.5f;
#pragma unroll
        for (int nt = 0; nt < NL; ++nt) {
            const float s = *reinterpret_cast<const float *>(img + col.s[nt]) * scale;
            acc[nt][0] = fmaf(s, e[nt][0], acc[nt][0]);
            acc[nt][1] = fmaf(s, e[nt][1], acc[nt][1]);
        }
    }
};
template <int P> struct MoeRecord<QT_Q8_0, P> : MoeRecordBlock<QT_Q8_0, P> {};
template <int P> struct MoeRecord<QT_Q4_0, P> : MoeRecordBlock<QT_Q4_0, P> {};
template <int P> struct MoeRecord<QT_MXFP4, P> : MoeRecordBlock<QT_MXFP4, P> {};

// The lane's columns of a group of n rows: columns beyond the last row repeat it (their sums are not stored)
template <int P, int NT> __device__ __forceinline__ MoeColumns<NT> moe_columns(int n, int lane) {
    constexpr int IMG = moe_image_bytes(P);
    const int g = lane >> 2, t = lane & 3;
    MoeColumns<NT> c;
    const int width = P == 2 && n * P <= 2 ? 2 : n * P <= 4 ? 4 : 8;      // columns of a class
    c.classes = 8 / width;
    c.class_b = g / width;
    c.class_s = 2 * t / width;
    const int gc = g % width, tc = 2 * t % width;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        c.b[nt] = min(nt * (8 / P) + gc / P, n - 1) * IMG + (gc % P) * 64 + t * 16;
        c.s[nt] = min(nt * (8 / P) + tc / P, n - 1) * IMG + P * 272 + 4 * (tc % P / 2);
    }
    c.row = c.class_s == 0 && tc % P == 0 ? tc / P : -1;
    return c;
}

// adds up a row's lanes: its plane pairs (P = 4) and classes
template <int P, int NT> __device__ __forceinline__ void moe_join(const MoeColumns<NT> &col, float (&acc)[NT][2]) {
    if (P == 4 || col.classes == 4) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[nt][i] += __shfl_xor_sync(0xFFFFFFFFu, acc[nt][i], 1);
    }
    if (col.classes >= 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[0][i] += __shfl_xor_sync(0xFFFFFFFFu, acc[0][i], 2);
    }
}

struct MoeHead {
    uint64_t full[kMoeMaxDepth];     // the producer's arrival and its copies' bytes
    uint64_t empty[kMoeMaxDepth];    // the eight warps
    MoeGroup group[kMoeMaxDepth];    // the stage's
    int fail;                        // some wait ran out: every role leaves its work
};

// one bounded wait of a role; on expiry (or when another role already gave up) the role leaves
__device__ __forceinline__ bool moe_wait(uint32_t bar, uint32_t parity, volatile int *fail, int *status) {
    if (mbar_try_wait_hint(bar, parity, 32)) return true;
    if (*fail) return false;
    if (mbar_wait_bounded_fast(bar, parity)) return true;
    atomicMax(status, DEV_ERR_PIPE_TIMEOUT);
    *fail = 1;
    return false;
}

// A product's part of one block: units (group, run of tiles) in turn, every unit's records a step at a time.  With `split` warps a tile
// (few tiles in all), a step takes as many records of 8 / split tiles, and the warps' sums are added up in order.
//   finish(unit's group, tile, slots, acc): one warp per tile; the lane holds the sums of rows g, g + 8 of slots[nt] (-1: of none)
template <int QT, int P, int NT, typename Finish> __device__ __forceinline__ void moe_product(const MoeProduct &p, uint8_t *smem, Finish finish) {
    constexpr int REC = moe_rec_bytes(QT), D = moe_depth(QT, P, NT), IMG = moe_image_bytes(P), kGroup = moe_group_rows(P, NT);
    __shared__ MoeHead head;
    __shared__ __align__(16) uint8_t zero[256 * P];
    __shared__ float part[NT == 1 ? 2 : 1][NT == 1 ? kMoeWarps : 1][2][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = NT == 1 ? p.split : 1, per = kMoeWarps / split;
    const int runs = (p.tiles + per - 1) / per, units = *p.lists.ngroups * runs, steps = (p.nrec + split - 1) / split;
    const int stage_bytes = moe_stage_bytes(QT, P, NT, split);
    volatile int *fail = &head.fail;
    if (tid == 0) {
        for (int i = 0; i < D; ++i) {
            mbar_init(smem_u32(&head.full[i]), 1);
            mbar_init(smem_u32(&head.empty[i]), kMoeWarps);
        }
        head.fail = 0;
        mbar_fence_init();
        fence_proxy_async();
    }
    for (int i = tid; i < 64 * P; i += kMoeThreads) reinterpret_cast<uint32_t *>(zero)[i] = 0u;
    __syncthreads();

    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    if (warp == kMoeWarps) {
        // ===== producer ==================================================================================
        bool full_ring = false;
        for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
            const int gi = u / runs, tile0 = (u - gi * runs) * per, tiles = min(per, p.tiles - tile0);
            const int word = lane < (int)(sizeof(MoeGroup) / 4) ? reinterpret_cast<const int *>(p.lists.groups + gi)[lane] : 0;
            const int expert = __shfl_sync(0xFFFFFFFFu, word, 0), n = __shfl_sync(0xFFFFFFFFu, word, 1);
            const uint8_t *w = p.w + expert * p.expert_bytes + (long long)tile0 * p.nrec * REC;
            const int slot = __shfl_sync(0xFFFFFFFFu, word, 2 + lane % 16);          // of row lane % 16
            const uint8_t *img = p.img + (size_t)(lane % 16 < n ? slot / p.slots_per_row : 0) * p.img_stride;
            for (int s = 0; s < steps; ++s) {
                if (full_ring) {
                    ok = __all_sync(0xFFFFFFFFu, moe_wait(smem_u32(&head.empty[stage]), phase ^ 1, fail, p.status));
                    if (!ok) break;
                }
                const int recs = min(split, p.nrec - s * split);
                const uint32_t bar = smem_u32(&head.full[stage]), dst = smem_u32(smem + stage * stage_bytes);
                if (lane < (int)(sizeof(MoeGroup) / 4)) reinterpret_cast<int *>(&head.group[stage])[lane] = word;
                fence_proxy_async();         // the readers' last accesses precede the copies
                __syncwarp();
                if (lane == 0) mbar_expect_tx(bar, recs * (tiles * REC + n * IMG));
                __syncwarp();
                if (lane < kMoeWarps) {      // warp lane's record
                    const int t = lane / split, r = lane % split;
                    if (t < tiles && r < recs) bulk_g2s(dst + lane * REC, w + ((long long)t * p.nrec + s * split + r) * REC, REC, bar);
                }
                if (lane % 16 < n)           // row lane % 16 of the group, every other record
                    for (int r = lane / 16; r < recs; r += 2)
                        bulk_g2s(dst + kMoeWarps * REC + (r * kGroup + lane % 16) * IMG, img + (size_t)(s * split + r) * IMG, IMG, bar);
                if (++stage == D) stage = 0, phase ^= 1, full_ring = true;
            }
        }
    } else {
        // ===== products ===================================================================================
        const int ws = warp % split, wt = warp / split;     // the warp's record of a step and tile of a unit
        int turn = 0;
        for (int u = blockIdx.x; u < units; u += gridDim.x) {
            const int gi = u / runs, tile = (u - gi * runs) * per + wt;
            MoeGroup grp;
            float acc[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = 0.f;
            // after a failure the products are left out, but the warps still meet
            ok = ok && __all_sync(0xFFFFFFFFu, moe_wait(smem_u32(&head.full[stage]), phase, fail, p.status));
            grp.expert = ok ? head.group[stage].expert : 0;
            grp.n = ok ? head.group[stage].n : 0;
            const int n = __shfl_sync(0xFFFFFFFFu, grp.n, 0);
            const MoeColumns<NT> col = moe_columns<P, NT>(max(n, 1), lane);
            int slot[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int r = nt * (8 / P) + col.row;
                slot[nt] = ok && col.row >= 0 && r < n ? head.group[stage].slot[r] : -1;
            }
            auto work = [&](auto mode) {
                for (int s = 0; s < steps; ++s) {
                    if (s > 0) ok = ok && __all_sync(0xFFFFFFFFu, moe_wait(smem_u32(&head.full[stage]), phase, fail, p.status));
                    if (!ok) break;
                    const uint8_t *at = smem + stage * stage_bytes;
                    if (tile < p.tiles && s * split + ws < p.nrec)
                        MoeRecord<QT, P>::template run<decltype(mode)>(at + warp * REC, lane, at + kMoeWarps * REC + ws * kGroup * IMG, zero, col, acc);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&head.empty[stage]));
                    if (++stage == D) stage = 0, phase ^= 1;
                }
            };
            const int used = n * P;              // columns
            if (P == 2 && used <= 2) work(MoeMode<1, 4>{});
            else if (used <= 4) work(MoeMode<1, 2>{});
            else if (used <= 8 || NT == 1) work(MoeMode<1, 1>{});
            else if (used <= 16) work(MoeMode<NT == 1 ? 1 : 2, 1>{});
            else work(MoeMode<NT, 1>{});
            moe_join<P, NT>(col, acc);
            if (NT == 1 && split > 1) {
                part[turn][warp][0][lane] = acc[0][0];
                part[turn][warp][1][lane] = acc[0][1];
                // a tile's warps meet.  (The next unit's sums go to the other half; that half's readers have met here since.)
                asm volatile("bar.sync %0, %1;" ::"r"(1 + wt), "r"(32 * split) : "memory");
                if (ws == 0)
                    for (int k = 1; k < split; ++k) acc[0][0] += part[turn][warp + k][0][lane], acc[0][1] += part[turn][warp + k][1][lane];
                turn ^= 1;
            }
            if (ok && ws == 0 && tile < p.tiles) finish(grp, tile, slot, acc);
        }
    }
    // After a failure copies may still be on their way: they get time to land (far above a copy's latency) before the block's
    // shared memory is released.
    __syncthreads();
    if (*fail) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 100000) {
        }
    }
}

// ---- gate, up and the activation function --------------------------------------------------------
template <int QT, int P, int NT>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_gate_up_kernel(const __grid_constant__ MoeGateUp p) {
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, g = lane >> 2;
    pdl_launch_dependents();
    pdl_wait();
    moe_product<QT, P, NT>(p.product, smem, [&](const MoeGroup &grp, int tile, const int (&slot)[NT], const float (&acc)[NT][2]) {
        const int f = tile * 8 + g;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (f >= p.ff || slot[nt] < 0) continue;
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
            p.h[(long long)slot[nt] * p.ff + f] = h;
        }
    });
}

// ---- down ------------------------------------------------------------------------------------------
template <int QT, int P, int NT>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_down_kernel(const __grid_constant__ MoeDown p) {
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, g = lane >> 2;
    pdl_launch_dependents();
    pdl_wait();
    moe_product<QT, P, NT>(p.product, smem, [&](const MoeGroup &grp, int tile, const int (&slot)[NT], const float (&acc)[NT][2]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (slot[nt] < 0) continue;
            float *z = p.z + (long long)slot[nt] * p.ld_z + tile * 16 + g;
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
    cudaError_t moe_wait_limit_##NAME(unsigned long long ns) { return cudaMemcpyToSymbol(s_wait_limit_ns, &ns, sizeof(ns)); }            \
    }
