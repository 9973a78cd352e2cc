// Low-rank adapters of many requests beside a shared projection: y[m] += scale * B (A x[m]) with the adapter that row m picks.
//
// One launch.  A cluster of eight blocks owns a few rows of one adapter: its blocks split K for t = A x, add their parts up through
// distributed shared memory in the order of the blocks, and split N for y += scale * B t.  So t never leaves the SMs, an adapter
// is read once per cluster, and no launch or device-wide wait stands between the two products.
//   * up to kLeaderRows rows (sequences decoding together, in any order): the cluster of row i counts the rows before it that have the same
//     adapter; every sixteenth leads a cluster of the next sixteen of them, the others' clusters end at once.  No list has to be
//     made first, and the grouping depends on the choices alone.
//   * more rows (prompts: long runs of one adapter): a cluster owns 32 neighbouring rows and takes the adapters that occur among
//     them one after the other.
// Both products run on mma.sync.m16n8k16 with bf16 operands and fp32 sums, the rows as M.  Operands of more bits are cut into
// bf16 planes: fp32 activations three (exact), fp16 adapters two (exact), t three where y is fp32 (exact) and two where y
// is rounded to bf16 anyway (an error of at most 2^-15 of t).  The adapters are kept in fragment order, so a load is 512 bytes a warp.
#include <cooperative_groups.h>

#include <algorithm>

#include "adapters.h"

namespace b200q {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = 8, kCluster = 8;
constexpr int kLeaderRows = 512, kTileRows = 32;

// D += A (16 x 16 bf16, row) * B (16 x 8 bf16, col)
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// two fp32 values as bf16 planes, upper bits first: truncation leaves a rest that the next plane takes
__device__ __forceinline__ uint32_t take_plane(float &a, float &b) {
    const uint32_t ua = __float_as_uint(a) & 0xFFFF0000u, ub = __float_as_uint(b) & 0xFFFF0000u;
    a -= __uint_as_float(ua);
    b -= __uint_as_float(ub);
    return __byte_perm(ua, ub, 0x7632);
}
__device__ __forceinline__ uint32_t last_plane(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <int PLANES> __device__ __forceinline__ void split(float a, float b, uint32_t (&out)[PLANES]) {
#pragma unroll
    for (int p = 0; p + 1 < PLANES; ++p) out[p] = take_plane(a, b);
    out[PLANES - 1] = last_plane(a, b);
}
// a pair of adapter elements as planes
template <bool F16, int PLANES> __device__ __forceinline__ void adapter_planes(uint32_t v, uint32_t (&out)[PLANES]) {
    if (F16) {
        const __half2 h = *reinterpret_cast<const __half2 *>(&v);
        split<PLANES>(__low2float(h), __high2float(h), out);
    } else {
        out[0] = v;
    }
}

struct RowList {
    int row[kTileRows];          // -1: no row
};

// eight elements of an activation row from k0 on, loaded ahead; zeros beyond K and for missing rows
template <bool XF32> struct XPiece {
    uint4 w[XF32 ? 2 : 1];
    __device__ __forceinline__ void load(const AdaptersParams &p, int row, int k0, bool wanted) {
#pragma unroll
        for (int i = 0; i < (XF32 ? 2 : 1); ++i) w[i] = make_uint4(0, 0, 0, 0);
        if (row < 0 || !wanted) return;
        if (XF32) {
            const uint32_t *src = reinterpret_cast<const uint32_t *>(p.x) + row * p.ldx + k0;
            if (p.x_vec && k0 + 8 <= p.K) {
#pragma unroll
                for (int i = 0; i < (XF32 ? 2 : 1); ++i) w[i] = reinterpret_cast<const uint4 *>(src)[i];
            } else {
                uint32_t v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = k0 + i < p.K ? src[i] : 0u;
#pragma unroll
                for (int i = 0; i < (XF32 ? 2 : 1); ++i) w[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
        } else {
            const unsigned short *src = reinterpret_cast<const unsigned short *>(p.x) + row * p.ldx + k0;
            if (p.x_vec && k0 + 8 <= p.K) {
                w[0] = *reinterpret_cast<const uint4 *>(src);
            } else {
                uint32_t v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t lo = k0 + 2 * j < p.K ? src[2 * j] : 0u, hi = k0 + 2 * j + 1 < p.K ? src[2 * j + 1] : 0u;
                    v[j] = lo | hi << 16;
                }
                w[0] = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
    }
    // as planes of four words (pairs of elements)
    __device__ __forceinline__ void planes(uint32_t (&out)[XF32 ? 3 : 1][4]) const {
        if (XF32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t v[XF32 ? 3 : 1];
                const uint4 &p = w[XF32 ? j >> 1 : 0];
                split(__uint_as_float(word_of(p, 2 * (j & 1))), __uint_as_float(word_of(p, 2 * (j & 1) + 1)), v);
#pragma unroll
                for (int i = 0; i < (XF32 ? 3 : 1); ++i) out[i][j] = v[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) out[0][j] = word_of(w[0], j);
        }
    }
};

// Eight neighbouring outputs (16-byte aligned), loaded ahead and put back with scale * v added
template <bool YF32> struct OutputPiece {
    uint4 w[YF32 ? 2 : 1];
    __device__ __forceinline__ void load(const uint8_t *y) {
#pragma unroll
        for (int i = 0; i < (YF32 ? 2 : 1); ++i) w[i] = reinterpret_cast<const uint4 *>(y)[i];
    }
    __device__ __forceinline__ void add(uint8_t *y, float scale, const float (&v)[8]) const {
        uint4 *out = reinterpret_cast<uint4 *>(y);
        if (YF32) {
#pragma unroll
            for (int i = 0; i < (YF32 ? 2 : 1); ++i)
                out[i] = make_uint4(__float_as_uint(fmaf(scale, v[4 * i], __uint_as_float(w[i].x))), __float_as_uint(fmaf(scale, v[4 * i + 1], __uint_as_float(w[i].y))),
                                    __float_as_uint(fmaf(scale, v[4 * i + 2], __uint_as_float(w[i].z))), __float_as_uint(fmaf(scale, v[4 * i + 3], __uint_as_float(w[i].w))));
        } else {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = word_of(w[0], i);
                o[i] = last_plane(fmaf(scale, v[2 * i], __uint_as_float(u << 16)), fmaf(scale, v[2 * i + 1], __uint_as_float(u & 0xFFFF0000u)));
            }
            out[0] = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
};
// one output
template <bool YF32> __device__ __forceinline__ void add_y(const AdapterSet &s, int row, int n, float scale, float v) {
    if (YF32) {
        float *y = reinterpret_cast<float *>(s.y) + row * s.ldy + n;
        *y = fmaf(scale, v, *y);
    } else {
        __nv_bfloat16 *y = reinterpret_cast<__nv_bfloat16 *>(s.y) + row * s.ldy + n;
        *y = __float2bfloat16_rn(fmaf(scale, v, __bfloat162float(*y)));
    }
}

// Shared memory: the warps' sums of a rank block (later a 16 x 32 piece of outputs per warp), this block's t, t as operand fragments.
// kRanks: ranks whose sums a warp holds at a time.
constexpr int kTileLd = 33;
template <int MT> struct Smem {
    static constexpr int kRows = 16 * MT, kKWarps = kWarps / MT, kRanks = MT == 1 ? 32 : 64, kChunks = MT == 1 ? 1 : 4;
    static constexpr size_t kSums = size_t(kKWarps) * kRows * kRanks * 4 > size_t(kWarps) * 16 * kTileLd * 4 ? size_t(kKWarps) * kRows * kRanks * 4
                                                                                                          : size_t(kWarps) * 16 * kTileLd * 4;
    static size_t bytes(int rank_pad, int planes) { return kSums + size_t(kRows) * rank_pad * 4 + size_t(MT) * (rank_pad / 16) * planes * 512; }
};

__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// one adapter against the rows of `list`
template <bool F16, bool XF32, bool YF32, int MT>
__device__ __forceinline__ void adapter_pass(const AdaptersParams &p, const AdapterSet &s, int slot, const RowList &list, int rank_pad_max, uint8_t *smem) {
    using S = Smem<MT>;
    constexpr int PX = XF32 ? 3 : 1, PA = F16 ? 2 : 1, PT = YF32 ? 3 : 2, RT = S::kRanks / 8;
    cg::cluster_group cluster = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, part = (int)cluster.block_rank();
    const int rank = s.rank[slot], rt = (rank + 7) / 8, rk = (rank + 15) / 16, rank_pad = 16 * rk;
    float *sums = reinterpret_cast<float *>(smem);
    float *tpart = reinterpret_cast<float *>(smem + S::kSums);
    uint4 *frag = reinterpret_cast<uint4 *>(smem + S::kSums + (size_t)S::kRows * rank_pad_max * 4);
    const float scale = s.scale[slot];
    const uint4 *b = reinterpret_cast<const uint4 *>(s.b + slot * s.b_stride);
    const long long pieces = (s.nchunks + S::kChunks - 1) / S::kChunks;
    const int nc0 = (int)(pieces * part / kCluster) * S::kChunks, nc1 = min((int)(pieces * (part + 1) / kCluster) * S::kChunks, s.nchunks);
    if (MT == 1)                             // B and y start their way while A is multiplied: 128 bytes a thread and turn
        for (long long i = (long long)nc0 * rk * 1024 + threadIdx.x * 128, end = min((long long)nc1 * rk * 1024, i + 64 * 1024); i < end; i += kThreads * 128)
            prefetch_l2(reinterpret_cast<const uint8_t *>(b) + i);

    // ---- t = A x over this block's part of K
    const int mt = warp % MT, kw = warp / MT;
    const int row0 = list.row[mt * 16 + g], row1 = list.row[mt * 16 + g + 8];
    const uint4 *a = reinterpret_cast<const uint4 *>(s.a + slot * s.a_stride);
    const int kc0 = (int)((long long)p.kchunks * part / kCluster), kc1 = (int)((long long)p.kchunks * (part + 1) / kCluster);
    for (int rb = 0; rb < rt; rb += RT) {
        const int tiles = min(rt - rb, RT);
        float acc[RT][4];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
        XPiece<XF32> x0, x1;                 // the next chunk's, on their way
        x0.load(p, row0, (kc0 + kw) * 32 + 8 * t, kc0 + kw < kc1);
        x1.load(p, row1, (kc0 + kw) * 32 + 8 * t, kc0 + kw < kc1);
        for (int kc = kc0 + kw; kc < kc1; kc += S::kKWarps) {
            uint32_t f0[PX][4], f1[PX][4];
            x0.planes(f0);
            x1.planes(f1);
            uint4 w[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i)
                if (i < tiles) w[i] = a[((size_t)kc * rt + rb + i) * 32 + lane];
            x0.load(p, row0, (kc + S::kKWarps) * 32 + 8 * t, kc + S::kKWarps < kc1);
            x1.load(p, row1, (kc + S::kKWarps) * 32 + 8 * t, kc + S::kKWarps < kc1);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                if (i >= tiles) break;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t b0[PA], b1[PA];
                    adapter_planes<F16, PA>(h ? w[i].z : w[i].x, b0);
                    adapter_planes<F16, PA>(h ? w[i].w : w[i].y, b1);
#pragma unroll
                    for (int px = 0; px < PX; ++px)
#pragma unroll
                        for (int pa = 0; pa < PA; ++pa)
                            mma_bf16(acc[i], f0[px][2 * h], f1[px][2 * h], f0[px][2 * h + 1], f1[px][2 * h + 1], b0[pa], b1[pa]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (i >= tiles) break;
            float *dst = sums + ((size_t)kw * S::kRows + mt * 16 + g) * S::kRanks + 8 * i + 2 * t;
            *reinterpret_cast<float2 *>(dst) = make_float2(acc[i][0], acc[i][1]);
            *reinterpret_cast<float2 *>(dst + 8 * S::kRanks) = make_float2(acc[i][2], acc[i][3]);
        }
        __syncthreads();
        const int width = min(rank_pad - 8 * rb, S::kRanks);        // the last tile of 16 may be half there
        for (int i = threadIdx.x; i < S::kRows * width; i += kThreads) {
            const int r = i / width, c = i - r * width;
            float v = 0.f;
            if (c < 8 * tiles)
#pragma unroll
                for (int w = 0; w < S::kKWarps; ++w) v += sums[((size_t)w * S::kRows + r) * S::kRanks + c];
            tpart[r * rank_pad + 8 * rb + c] = v;
        }
        __syncthreads();
    }
    cluster.sync();

    // ---- t over all of K, as operand fragments: [row tile][rank tile][plane][lane]
    for (int i = threadIdx.x; i < MT * rk * 32; i += kThreads) {
        const int l = i & 31, tile = i >> 5, m = tile / rk, k = tile - m * rk;
        uint32_t w[4][PT];
#pragma unroll
        for (int e = 0; e < 4; ++e) {                            // (row g, ranks 2 t), (row g + 8, ..), (row g, ranks 2 t + 8), (..)
            const int at = (m * 16 + (l >> 2) + 8 * (e & 1)) * rank_pad + k * 16 + 2 * (l & 3) + 8 * (e >> 1);
            float2 o[kCluster], v = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < kCluster; ++c) o[c] = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(tpart, c) + at);
#pragma unroll
            for (int c = 0; c < kCluster; ++c) v.x += o[c].x, v.y += o[c].y;
            split<PT>(v.x, v.y, w[e]);
        }
#pragma unroll
        for (int q = 0; q < PT; ++q) frag[((size_t)tile * PT + q) * 32 + l] = make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
    }
    __syncthreads();
    auto arrived = cluster.barrier_arrive();                      // this block has read the others' parts

    // ---- y += scale B t over this block's part of N
    // acc of column tile i: rows g, g + 8 of row tile m, outputs 8 t + 2 i, + 1 of the chunk
    auto multiply = [&](int nc, int m, float (&acc)[4][4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
        const uint4 *bp = b + (size_t)nc * rk * 64 + lane, *fp = frag + (size_t)m * rk * PT * 32 + lane;
#pragma unroll 2
        for (int k = 0; k < rk; ++k, bp += 64, fp += PT * 32) {
            const uint4 w[2] = {bp[0], bp[32]};
            uint4 f[PT];
#pragma unroll
            for (int q = 0; q < PT; ++q) f[q] = fp[q * 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t b0[PA], b1[PA];
                adapter_planes<F16, PA>(i & 1 ? w[i >> 1].z : w[i >> 1].x, b0);
                adapter_planes<F16, PA>(i & 1 ? w[i >> 1].w : w[i >> 1].y, b1);
#pragma unroll
                for (int q = 0; q < PT; ++q)
#pragma unroll
                    for (int pa = 0; pa < PA; ++pa) mma_bf16(acc[i], f[q].x, f[q].y, f[q].z, f[q].w, b0[pa], b1[pa]);
            }
        }
    };
    // Warps share the row tiles and the chunks; with many rows a warp takes four neighbouring chunks of sixteen rows at a time: whole
    // 256-byte pieces of bf16 rows.
    constexpr int CH = S::kChunks, kStep = S::kKWarps * CH;
    const int m = warp % MT;
    int nc = nc0 + (warp / MT) * CH;
    if (s.y_vec) {
        constexpr int YB = YF32 ? 4 : 2;
        const int r0 = list.row[m * 16 + g], r1 = list.row[m * 16 + g + 8];
        uint8_t *row[2] = {reinterpret_cast<uint8_t *>(s.y) + (r0 * s.ldy + nc * 32 + 8 * t) * YB, reinterpret_cast<uint8_t *>(s.y) + (r1 * s.ldy + nc * 32 + 8 * t) * YB};
        const bool have[2] = {r0 >= 0, r1 >= 0};
        for (; nc + CH <= nc1 && (nc + CH) * 32 <= s.n; nc += kStep) {
            OutputPiece<YF32> y[CH][2];
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (have[h]) y[c][h].load(row[h] + c * 32 * YB);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float acc[4][4];
                multiply(nc + c, m, acc);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[2 * i] = acc[i][2 * h], v[2 * i + 1] = acc[i][2 * h + 1];
                    if (have[h]) y[c][h].add(row[h] + c * 32 * YB, scale, v);
                }
            }
            row[0] += kStep * 32 * YB;
            row[1] += kStep * 32 * YB;
        }
    }
    // rows that are not aligned, the last outputs: a row's 32 by 32 lanes
    float *piece = sums + warp * 16 * kTileLd;
    for (; nc < nc1; nc += kStep)
#pragma unroll 1
        for (int c = nc; c < min(nc + CH, nc1); ++c) {
            float acc[4][4];
            multiply(c, m, acc);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) piece[(g + 8 * (j >> 1)) * kTileLd + 8 * t + 2 * i + (j & 1)] = acc[i][j];
            __syncwarp();
            if (c * 32 + lane < s.n)
#pragma unroll 8
                for (int r = 0; r < 16; ++r) {
                    const int to = list.row[m * 16 + r];
                    if (to >= 0) add_y<YF32>(s, to, c * 32 + lane, scale, piece[r * kTileLd + lane]);
                }
        }
    cluster.barrier_wait(std::move(arrived));
}

template <bool F16, bool XF32, bool YF32, int MT>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, MT == 1 && !XF32 && !F16 ? 3 : 2) adapters_kernel(const __grid_constant__ AdaptersParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ RowList list;
    __shared__ int s_slot[kTileRows];
    __shared__ int s_count[kWarps];
    const AdapterSet &s = p.set[blockIdx.y];
    const int id = blockIdx.x / kCluster, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    pdl_wait();
    // an adapter that takes part: within the set and loaded
    auto active = [&](int slot) { return (unsigned)slot < (unsigned)s.slots && s.rank[slot] > 0; };
    // (every block of a cluster sees the same rows and takes the same way)
    if (MT == 1) {
        const int slot = p.rows[id];
        if (!active(slot)) return;
        int before = 0;
        for (int i = tid; i < id; i += kThreads) before += p.rows[i] == slot;
        before = __reduce_add_sync(0xFFFFFFFFu, before);
        if (lane == 0) s_count[warp] = before;
        if (tid < kTileRows) list.row[tid] = -1;
        __syncthreads();
        before = 0;
        for (int w = 0; w < kWarps; ++w) before += s_count[w];
        if (before % 16) return;
        if (warp == 0) {
            int found = 0;
            for (int i0 = id; i0 < p.m && found < 16; i0 += 32) {
                const bool mine = i0 + lane < p.m && p.rows[i0 + lane] == slot;
                const unsigned all = __ballot_sync(0xFFFFFFFFu, mine);
                const int at = found + __popc(all & ((1u << lane) - 1));
                if (mine && at < 16) list.row[at] = i0 + lane;
                found += __popc(all);
            }
        }
        __syncthreads();
        adapter_pass<F16, XF32, YF32, MT>(p, s, slot, list, p.rank_pad, smem);
    } else {
        static_assert(MT <= 2, "one warp looks the rows over");
        const int base = id * kTileRows;
        if (warp == 0) {
            int slot = base + lane < p.m ? p.rows[base + lane] : -1;
            if (!active(slot)) slot = -1;
            s_slot[lane] = slot;
            const unsigned same = __match_any_sync(0xFFFFFFFFu, slot);      // (all lanes take part, rows without an adapter too)
            const unsigned first = __ballot_sync(0xFFFFFFFFu, slot >= 0 && __ffs(same) - 1 == lane);
            if (lane == 0) s_count[0] = (int)first;
        }
        __syncthreads();
        for (unsigned left = (unsigned)s_count[0]; left; left &= left - 1) {      // the rows that are the first of their adapter
            const int slot = s_slot[__ffs((int)left) - 1];
            if (tid < kTileRows) list.row[tid] = s_slot[tid] == slot ? base + tid : -1;
            __syncthreads();
            adapter_pass<F16, XF32, YF32, MT>(p, s, slot, list, p.rank_pad, smem);
            __syncthreads();
        }
    }
}

template <bool F16, bool XF32, bool YF32, int MT> cudaError_t launch(const AdaptersParams &p, int clusters, cudaStream_t st) {
    auto kern = adapters_kernel<F16, XF32, YF32, MT>;
    const size_t smem = Smem<MT>::bytes(p.rank_pad, YF32 ? 3 : 2);
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(clusters * kCluster), (unsigned)p.sets);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

template <bool F16, bool XF32, bool YF32> cudaError_t launch_rows(const AdaptersParams &p, cudaStream_t st) {
    if (p.m <= kLeaderRows) return launch<F16, XF32, YF32, 1>(p, p.m, st);
    return launch<F16, XF32, YF32, kTileRows / 16>(p, (p.m + kTileRows - 1) / kTileRows, st);
}

// A[rank][K], B[N][rank] (row-major) -> fragments
__global__ void adapter_pack_kernel(const uint16_t *a, const uint16_t *b, uint4 *pa, uint4 *pb, int rank, int K, int n, int kchunks, int nchunks) {
    const int rt = (rank + 7) / 8, rk = (rank + 15) / 16;
    const long long na = (long long)kchunks * rt * 32, nb = (long long)nchunks * rk * 64;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < na + nb; i += (long long)gridDim.x * blockDim.x) {
        const int lane = (int)(i & 31), g = lane >> 2, t = lane & 3;
        uint32_t w[4] = {0, 0, 0, 0};
        if (i < na) {                    // rank 8 tile + g, k = 32 chunk + 8 t .. + 7
            const long long c = i >> 5;
            const int r = (int)(c % rt) * 8 + g, k = (int)(c / rt) * 32 + 8 * t;
            for (int j = 0; j < 8; ++j)
                if (r < rank && k + j < K) w[j >> 1] |= (uint32_t)a[(long long)r * K + k + j] << (16 * (j & 1));
            pa[i] = make_uint4(w[0], w[1], w[2], w[3]);
        } else {                         // two of the chunk's four column tiles: column g of tile v is n = 32 chunk + 8 (g / 2) + 2 v + g % 2
            const long long c = (i - na) >> 5;
            const int v = (int)(c & 1) * 2, k = (int)((c >> 1) % rk) * 16 + 2 * t;
            for (int j = 0; j < 8; ++j) {
                const int col = (int)((c >> 1) / rk) * 32 + 8 * (g >> 1) + 2 * (v + (j >> 2)) + (g & 1), r = k + 8 * ((j >> 1) & 1) + (j & 1);
                if (col < n && r < rank) w[j >> 1] |= (uint32_t)b[(long long)col * rank + r] << (16 * (j & 1));
            }
            pb[i - na] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

}  // namespace

cudaError_t adapter_pack(const void *a, const void *b, uint8_t *pa, uint8_t *pb, int rank, int K, int n, cudaStream_t st) {
    const int kchunks = (K + 31) / 32, nchunks = (n + 31) / 32;
    adapter_pack_kernel<<<512, 256, 0, st>>>((const uint16_t *)a, (const uint16_t *)b, reinterpret_cast<uint4 *>(pa), reinterpret_cast<uint4 *>(pb), rank, K, n,
                                             kchunks, nchunks);
    return cudaGetLastError();
}

cudaError_t adapters_run(const AdaptersParams &p, bool f16, bool x_f32, bool y_f32, cudaStream_t st) {
    if (f16) return x_f32 ? (y_f32 ? launch_rows<true, true, true>(p, st) : launch_rows<true, true, false>(p, st))
                          : (y_f32 ? launch_rows<true, false, true>(p, st) : launch_rows<true, false, false>(p, st));
    return x_f32 ? (y_f32 ? launch_rows<false, true, true>(p, st) : launch_rows<false, true, false>(p, st))
                 : (y_f32 ? launch_rows<false, false, true>(p, st) : launch_rows<false, false, false>(p, st));
}

}  // namespace b200q
