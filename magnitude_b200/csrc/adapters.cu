// Low-rank adapters of many requests beside a shared projection: y[m] += scale * B (A x[m]) with the adapter that row m picks.
//
//   * up to kFewRows rows (sequences decoding together, in any order, or the pieces of a few prompts): one launch of clusters of eight blocks.
//     A cluster takes up to sixteen rows of one adapter and one projection at a time; its blocks split K for t = A x, add their parts
//     up through distributed shared memory in the order of the blocks, and split N for y += scale * B t, so t never leaves the SMs.
//     Every block finds the rows of each adapter for itself.
//   * more rows (long runs of one adapter): two launches, t = A x for tiles of 32 rows (K cut into a few ranges to fill the chip), then
//     y += scale * B t as one stream over y.  A tile takes the adapters that occur among its rows one after the other.
// Both products run on mma.sync.m16n8k16 with bf16 operands and fp32 sums, the rows as M.  Operands of more bits are cut into
// bf16 planes: fp32 activations three (exact), fp16 adapters two (exact), t three where y is fp32 (exact) and two where y
// is rounded to bf16 anyway (an error of at most 2^-15 of t).  The adapters are kept in fragment order, so a load is 512 bytes a warp.
#include <cooperative_groups.h>

#include <algorithm>

#include "adapters.h"
#include "launch.h"

namespace b200q {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = 8, kCluster = 8;
constexpr int kFewRows = 512;

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

// eight elements of an activation row from k0 on, loaded ahead; zeros beyond K and for missing rows
template <bool XF32> struct XPiece {
    uint4 w[XF32 ? 2 : 1];
    __device__ __forceinline__ void load(const AdaptersParams &p, long long row, int k0, bool wanted) {
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
template <bool YF32> __device__ __forceinline__ float load_y(const AdapterSet &s, long long row, int n) {
    if (YF32) return reinterpret_cast<const float *>(s.y)[row * s.ldy + n];
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(s.y)[row * s.ldy + n]);
}
template <bool YF32> __device__ __forceinline__ void store_y(const AdapterSet &s, long long row, int n, float v) {
    if (YF32) reinterpret_cast<float *>(s.y)[row * s.ldy + n] = v;
    else reinterpret_cast<__nv_bfloat16 *>(s.y)[row * s.ldy + n] = __float2bfloat16_rn(v);
}

// acc += sixteen rows (planes of eight elements of rows g, g + 8) times a fragment of A: 32 of K, eight ranks
template <bool F16, int PX> __device__ __forceinline__ void multiply_tile(const uint32_t (&f0)[PX][4], const uint32_t (&f1)[PX][4], const uint4 &w, float (&acc)[4]) {
    constexpr int PA = F16 ? 2 : 1;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t b0[PA], b1[PA];
        adapter_planes<F16, PA>(h ? w.z : w.x, b0);
        adapter_planes<F16, PA>(h ? w.w : w.y, b1);
#pragma unroll
        for (int px = 0; px < PX; ++px)
#pragma unroll
            for (int pa = 0; pa < PA; ++pa) mma_bf16(acc, f0[px][2 * h], f1[px][2 * h], f0[px][2 * h + 1], f1[px][2 * h + 1], b0[pa], b1[pa]);
    }
}

// acc += a piece of t = A x for sixteen rows: tiles of eight ranks, chunks kc, kc + step, .. below kc1.  r0, r1: the lane's rows, -1: none;
// w(i, kc): the lane's fragment of tile i.
template <bool F16, bool XF32, int RT, typename Fragment>
__device__ __forceinline__ void shrink(const AdaptersParams &p, long long r0, long long r1, int kc, int kc1, int step, int tiles, int t, Fragment fragment, float (&acc)[RT][4]) {
    constexpr int PX = XF32 ? 3 : 1;
    XPiece<XF32> x0, x1;                     // the next chunk's, on their way
    x0.load(p, r0, kc * 32 + 8 * t, kc < kc1);
    x1.load(p, r1, kc * 32 + 8 * t, kc < kc1);
    for (; kc < kc1; kc += step) {
        uint32_t f0[PX][4], f1[PX][4];
        x0.planes(f0);
        x1.planes(f1);
        uint4 w[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i)
            if (i < tiles) w[i] = fragment(i, kc);
        x0.load(p, r0, (kc + step) * 32 + 8 * t, kc + step < kc1);
        x1.load(p, r1, (kc + step) * 32 + 8 * t, kc + step < kc1);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (i >= tiles) break;
            multiply_tile<F16, PX>(f0, f1, w[i], acc[i]);
        }
    }
}

// B t of sixteen rows and a chunk of 32 outputs: acc of column tile i: rows g, g + 8, outputs 8 t + 2 i, + 1.  bp: the lane's fragments of the
// chunk, fp: of the rows' t
template <bool F16, int PT> __device__ __forceinline__ void expand(const uint4 *bp, const uint4 *fp, int rk, float (&acc)[4][4]) {
    constexpr int PA = F16 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
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
}

// y of sixteen rows += scale B t over the chunks nc, nc + step, .. below nc1, CH neighbouring ones at a time.  row[16]: the rows, -1: none;
// piece: 16 x kTileLd floats of the warp
constexpr int kTileLd = 33;
template <bool F16, bool YF32, int CH>
__device__ __forceinline__ void add_chunks(const AdapterSet &s, const uint4 *b, const uint4 *frag, int rk, float scale, const int *row, int nc, int nc1, int step, float *piece,
                                           int lane) {
    constexpr int PT = YF32 ? 3 : 2, YB = YF32 ? 4 : 2;
    const int g = lane >> 2, t = lane & 3;
    if (s.y_vec) {
        const int r0 = row[g], r1 = row[g + 8];
        uint8_t *to[2] = {reinterpret_cast<uint8_t *>(s.y) + (r0 * s.ldy + nc * 32 + 8 * t) * YB, reinterpret_cast<uint8_t *>(s.y) + (r1 * s.ldy + nc * 32 + 8 * t) * YB};
        for (; nc + CH <= nc1 && (nc + CH) * 32 <= s.n; nc += step) {
            OutputPiece<YF32> y[CH][2];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (r0 >= 0) y[c][0].load(to[0] + c * 32 * YB);
                if (r1 >= 0) y[c][1].load(to[1] + c * 32 * YB);
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float acc[4][4];
                expand<F16, PT>(b + (size_t)(nc + c) * rk * 64 + lane, frag + lane, rk, acc);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[2 * i] = acc[i][2 * h], v[2 * i + 1] = acc[i][2 * h + 1];
                    if ((h ? r1 : r0) >= 0) y[c][h].add(to[h] + c * 32 * YB, scale, v);
                }
            }
            to[0] += step * 32 * YB;
            to[1] += step * 32 * YB;
        }
    }
    // rows that are not aligned, the last outputs: a row's 32 by 32 lanes
    for (; nc < nc1; nc += step)
#pragma unroll 1
        for (int c = nc; c < min(nc + CH, nc1); ++c) {
            float acc[4][4];
            expand<F16, PT>(b + (size_t)c * rk * 64 + lane, frag + lane, rk, acc);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) piece[(g + 8 * (j >> 1)) * kTileLd + 8 * t + 2 * i + (j & 1)] = acc[i][j];
            __syncwarp();
            if (c * 32 + lane < s.n)
#pragma unroll
                for (int r0 = 0; r0 < 16; r0 += 8) {         // eight loads, then eight stores
                    float old[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) old[r] = row[r0 + r] >= 0 ? load_y<YF32>(s, row[r0 + r], c * 32 + lane) : 0.f;
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (row[r0 + r] >= 0) store_y<YF32>(s, row[r0 + r], c * 32 + lane, fmaf(scale, piece[(r0 + r) * kTileLd + lane], old[r]));
                }
        }
}

// an adapter that takes part: within the set and loaded
__device__ __forceinline__ bool active(const AdapterSet &s, int slot) { return (unsigned)slot < (unsigned)s.slots && s.rank[slot] > 0; }

// ---- up to kFewRows rows ---------------------------------------------------------------------------------

// The rows by adapter: groups of up to sixteen, adapters in the order of their first rows.  Warp w owns rows 64 w .. 64 w + 63.
constexpr int kKeys = 2 * kFewRows;
struct FewRows {
    int slot[kFewRows];
    int key[kKeys];                                  // a table of the slots that occur: open addressing
    int first_row[kKeys];                            // of every key
    short row_base[kKeys], group_base[kKeys];        // where its rows, its groups begin
    uint8_t count[kWarps][kKeys];                    // its rows in every warp
    short sorted[kFewRows], first[kFewRows + 1];     // rows of group i: sorted[first[i]] .. sorted[first[i + 1] - 1]
    int2 sums[kWarps];
    int n;
};
__device__ __forceinline__ void few_groups(FewRows &l, const AdaptersParams &p) {
    static_assert(kFewRows == 64 * kWarps, "rows of a warp");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (p.m == 1) {                                  // nothing to sort
        if (tid == 0) {
            l.slot[0] = p.rows[0];
            l.sorted[0] = l.first[0] = 0;
            l.first[1] = 1;
            l.n = 1;
        }
        __syncthreads();
        return;
    }
    for (int i = tid; i < kKeys; i += kThreads) {
        l.key[i] = -1;
        l.first_row[i] = kFewRows;
    }
    for (int i = tid; i < kWarps * kKeys / 4; i += kThreads) reinterpret_cast<uint32_t *>(l.count)[i] = 0u;
    __syncthreads();
    int at[2], rank[2];                              // key and place among the warp's rows of the same slot
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = warp * 64 + h * 32 + lane, slot = i < p.m ? p.rows[i] : -1;
        l.slot[i] = slot;
        at[h] = -1;
        if (slot >= 0) {
            int k = (int)(((unsigned)slot * 2654435761u) >> 22);      // (Fibonacci hashing: the upper ten bits)
            while (true) {
                const int old = atomicCAS(&l.key[k], -1, slot);
                if (old == -1 || old == slot) break;
                k = (k + 1) & (kKeys - 1);
            }
            at[h] = k;
            atomicMin(&l.first_row[k], i);
        }
        __syncwarp();
        const unsigned same = __match_any_sync(0xFFFFFFFFu, at[h]);
        const int before = at[h] >= 0 ? l.count[warp][at[h]] : 0;
        rank[h] = before + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (at[h] >= 0 && (same >> lane) == 1u) l.count[warp][at[h]] = (uint8_t)(rank[h] + 1);      // the last lane of those
        __syncwarp();
    }
    __syncthreads();
    int all[2];
    int2 mine = make_int2(0, 0), run[2];             // rows and groups that begin with this thread's rows
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        all[h] = 0;
        int before = 0;
        if (at[h] >= 0)
            for (int w = 0; w < kWarps; ++w) {
                const int n = l.count[w][at[h]];
                all[h] += n;
                before += w < warp ? n : 0;
            }
        rank[h] += before;
        const bool begins = at[h] >= 0 && l.first_row[at[h]] == warp * 64 + h * 32 + lane;
        run[h] = begins ? make_int2(all[h], (all[h] + 15) / 16) : make_int2(0, 0);
        const int2 own = run[h];
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int x = __shfl_up_sync(0xFFFFFFFFu, run[h].x, d), y = __shfl_up_sync(0xFFFFFFFFu, run[h].y, d);
            if (lane >= d) run[h].x += x, run[h].y += y;
        }
        const int2 sum = make_int2(__shfl_sync(0xFFFFFFFFu, run[h].x, 31), __shfl_sync(0xFFFFFFFFu, run[h].y, 31));
        run[h].x += mine.x - own.x, run[h].y += mine.y - own.y;
        mine.x += sum.x, mine.y += sum.y;
    }
    if (lane == 0) l.sums[warp] = mine;
    __syncthreads();
    int2 base = make_int2(0, 0), total = make_int2(0, 0);
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) base.x += l.sums[w].x, base.y += l.sums[w].y;
        total.x += l.sums[w].x, total.y += l.sums[w].y;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (at[h] >= 0 && l.first_row[at[h]] == warp * 64 + h * 32 + lane) {
            l.row_base[at[h]] = (short)(base.x + run[h].x);
            l.group_base[at[h]] = (short)(base.y + run[h].y);
        }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (at[h] >= 0) {
            const int to = l.row_base[at[h]] + rank[h];
            l.sorted[to] = (short)(warp * 64 + h * 32 + lane);
            if (rank[h] % 16 == 0) l.first[l.group_base[at[h]] + rank[h] / 16] = (short)to;
        }
    if (tid == 0) {
        l.n = total.y;
        l.first[total.y] = (short)total.x;
    }
    __syncthreads();
}

// Shared memory beside the rows: the warps' sums of a rank block (later a 16 x 32 piece of outputs each), this block's t, t as fragments
constexpr int kFewRanks = 32;                        // ranks whose sums a warp holds at a time
constexpr size_t kFewSums = size_t(kWarps) * 16 * kTileLd * 4;
static_assert(kFewSums >= size_t(kWarps) * 16 * kFewRanks * 4, "sums");
size_t few_smem(int rank_pad, int planes) { return kFewSums + size_t(16) * rank_pad * 4 + size_t(rank_pad / 16) * planes * 512; }

// the block's threads ask for a piece of memory, 128 bytes each and turn (at most 64 KB)
__device__ __forceinline__ void prefetch_bytes(const uint8_t *p, long long bytes) {
    for (int i = threadIdx.x * 128; i < min(bytes, 65536ll); i += kThreads * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + i));
}

// one adapter against up to sixteen rows
template <bool F16, bool XF32, bool YF32>
__device__ __forceinline__ void few_pass(const AdaptersParams &p, const AdapterSet &s, int slot, const int *row, int parts, uint8_t *smem) {
    constexpr int PT = YF32 ? 3 : 2, RT = kFewRanks / 8;
    cg::cluster_group cluster = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int block = (int)cluster.block_rank(), part = block & (parts - 1), lead = block - part;
    const int rank = slot < 0 ? 0 : s.rank[slot], rt = (rank + 7) / 8, rk = (rank + 15) / 16, rank_pad = 16 * rk;
    float *sums = reinterpret_cast<float *>(smem);
    float *tpart = reinterpret_cast<float *>(smem + kFewSums);
    uint4 *frag = reinterpret_cast<uint4 *>(smem + kFewSums + (size_t)16 * p.rank_pad * 4);
    const float scale = slot < 0 ? 0.f : s.scale[slot];
    const uint4 *a = reinterpret_cast<const uint4 *>(s.a + slot * s.a_stride), *b = reinterpret_cast<const uint4 *>(s.b + slot * s.b_stride);
    const int nc0 = (int)((long long)s.nchunks * part / parts), nc1 = slot < 0 ? nc0 : (int)((long long)s.nchunks * (part + 1) / parts);
    const int kc0 = (int)((long long)p.kchunks * part / parts), kc1 = (int)((long long)p.kchunks * (part + 1) / parts);
    // the block's parts of A (what is not read at once) and B all start their way
    prefetch_bytes(reinterpret_cast<const uint8_t *>(a) + (long long)(kc0 + kWarps) * rt * 512, (long long)(kc1 - kc0 - kWarps) * rt * 512);
    prefetch_bytes(reinterpret_cast<const uint8_t *>(b) + (long long)nc0 * rk * 1024, (long long)(nc1 - nc0) * rk * 1024);

    // ---- t = A x over this block's part of K
    for (int rb = 0; rb < rt; rb += RT) {
        const int tiles = min(rt - rb, RT);
        float acc[RT][4];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
        shrink<F16, XF32, RT>(p, row[g], row[g + 8], kc0 + warp, kc1, kWarps, tiles, t, [&](int i, int kc) { return a[((size_t)kc * rt + rb + i) * 32 + lane]; }, acc);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (i >= tiles) break;
            float *dst = sums + (warp * 16 + g) * kFewRanks + 8 * i + 2 * t;
            *reinterpret_cast<float2 *>(dst) = make_float2(acc[i][0], acc[i][1]);
            *reinterpret_cast<float2 *>(dst + 8 * kFewRanks) = make_float2(acc[i][2], acc[i][3]);
        }
        __syncthreads();
        const int width = min(rank_pad - 8 * rb, kFewRanks);        // the last tile of 16 may be half there
        for (int i = threadIdx.x; i < 16 * width; i += kThreads) {
            const int r = i / width, c = i - r * width;
            float v = 0.f;
            if (c < 8 * tiles)
#pragma unroll
                for (int w = 0; w < kWarps; ++w) v += sums[(w * 16 + r) * kFewRanks + c];
            tpart[r * rank_pad + 8 * rb + c] = v;
        }
        __syncthreads();
    }
    cluster.sync();

    // ---- t over all of K, as operand fragments: [rank tile][plane][lane]
    for (int i = threadIdx.x; i < rk * 32; i += kThreads) {
        const int l = i & 31, k = i >> 5;
        uint32_t w[4][PT];
#pragma unroll
        for (int e = 0; e < 4; ++e) {                            // (row g, ranks 2 t), (row g + 8, ..), (row g, ranks 2 t + 8), (..)
            const int at = ((l >> 2) + 8 * (e & 1)) * rank_pad + k * 16 + 2 * (l & 3) + 8 * (e >> 1);
            float2 o[kCluster], v = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < kCluster; ++c)
                if (c < parts) o[c] = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(tpart, lead + c) + at);
#pragma unroll
            for (int c = 0; c < kCluster; ++c)
                if (c < parts) v.x += o[c].x, v.y += o[c].y;
            split<PT>(v.x, v.y, w[e]);
        }
#pragma unroll
        for (int q = 0; q < PT; ++q) frag[((size_t)k * PT + q) * 32 + l] = make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
    }
    __syncthreads();
    auto arrived = cluster.barrier_arrive();                      // this block has read the others' parts

    // ---- y += scale B t over this block's part of N
    add_chunks<F16, YF32, 1>(s, b, frag, rk, scale, row, nc0 + warp, nc1, kWarps, sums + warp * 16 * kTileLd, lane);
    cluster.barrier_wait(std::move(arrived));
}

template <bool F16, bool XF32, bool YF32>
__global__ void __launch_bounds__(kThreads, 2) adapters_few_kernel(const __grid_constant__ AdaptersParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(16) FewRows rows;
    __shared__ int row[16];
    pdl_launch_dependents();
    pdl_wait();
    few_groups(rows, p);
    // As many blocks of a cluster share an item (a group and a set) as there are blocks for all items: eight of few, one of many.  (Every
    // block has the same groups; those of a cluster meet the same number of times.)
    const int items = rows.n * p.sets, block = (int)(blockIdx.x % kCluster);
    int parts = kCluster;
    while (parts > 1 && items * parts > (int)gridDim.x) parts /= 2;
    const int at_a_time = gridDim.x / parts, rounds = (items + at_a_time - 1) / at_a_time;
    for (int round = 0; round < rounds; ++round) {
        const int item = round * at_a_time + blockIdx.x / kCluster * (kCluster / parts) + block / parts;
        const int group = min(item, items - 1) / p.sets, set = min(item, items - 1) - group * p.sets;
        const AdapterSet &s = p.set[set];
        const int first = rows.first[group], n = rows.first[group + 1] - first;
        int slot = item < items ? rows.slot[rows.sorted[first]] : -1;
        if (!active(s, slot)) slot = -1;
        if (threadIdx.x < 16) row[threadIdx.x] = slot >= 0 && threadIdx.x < n ? rows.sorted[first + threadIdx.x] : -1;
        __syncthreads();
        few_pass<F16, XF32, YF32>(p, s, slot, row, parts, smem);
        __syncthreads();
    }
}

// ---- more rows ---------------------------------------------------------------------------------------------
// bit mask of the warp's lanes whose slot is the first of its kind
__device__ __forceinline__ unsigned first_rows(int slot, int lane) {
    const unsigned same = __match_any_sync(0xFFFFFFFFu, slot);      // (all lanes take part, rows without an adapter too)
    return __ballot_sync(0xFFFFFFFFu, slot >= 0 && __ffs(same) - 1 == lane);
}

// t[row][ranks of all sets].  A cluster takes 128 rows, sixteen a warp, and one adapter of them after the other; its blocks split K and add their
// parts up through distributed shared memory, each for some of the rows.  x and the fragments of A come into shared memory by cp.async, 512
// bytes of every row at a time.  (With x in registers, a chunk ahead, the way from L2 set the pace: 4096 rows of 5120, 64 ranks, 54 us.)
constexpr int kSumTiles = 8, kShrinkRows = 16 * kWarps;      // tiles of eight ranks whose sums a warp holds at a time
constexpr int kSumLd = 8 * kSumTiles + 2;
constexpr int kXLd = 512 + 64;                               // bytes from row to row: two rows' pieces lie in different banks
constexpr size_t kShrinkX = size_t(kShrinkRows) * kXLd;
__host__ __device__ constexpr int batch_chunks(bool f32) { return f32 ? 4 : 8; }
constexpr size_t kShrinkSmem = kShrinkX + size_t(8) * kSumTiles * 512;
static_assert(kShrinkX >= size_t(kShrinkRows) * kSumLd * 4, "sums");
struct AdapterTile {
    const uint4 *from;                   // its fragment of the first chunk
    int step, to;                        // 16-byte words from chunk to chunk; its place in a row of t
};
template <bool F16, bool XF32> __global__ void __launch_bounds__(kThreads, 2) adapters_shrink_kernel(const __grid_constant__ AdaptersParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int slots[kShrinkRows];
    __shared__ unsigned firsts[kShrinkRows / 32];
    __shared__ AdapterTile tiles_of[kAdapterMaxSets * kAdapterMaxRank / 8];
    __shared__ int all_tiles;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int base = blockIdx.x * kShrinkRows, mine = warp * 16;
    const int parts = gridDim.y, part0 = blockIdx.y;      // the cluster
    const int kc0 = (int)((long long)p.kchunks * part0 / parts), kc1 = (int)((long long)p.kchunks * (part0 + 1) / parts);
    cg::cluster_group cluster = cg::this_cluster();
    float *sums = reinterpret_cast<float *>(smem);        // [row][rank of the tiles at hand], where x was
    uint8_t *afrag = smem + kShrinkX;
    constexpr int PX = XF32 ? 3 : 1, XB = XF32 ? 4 : 2, BATCH = batch_chunks(XF32);
    pdl_launch_dependents();
    pdl_wait();
    if (tid < kShrinkRows) {
        const int slot = base + tid < p.m ? p.rows[base + tid] : -1;
        slots[tid] = slot;
        const unsigned first = first_rows(slot, lane);
        if (lane == 0) firsts[warp] = first;
    }
    __syncthreads();
    for (int part = 0; part < kShrinkRows / 32; ++part)
        for (unsigned left = firsts[part]; left; left &= left - 1) {
            const int slot = slots[part * 32 + __ffs((int)left) - 1];
            bool seen = false;               // had its turn among earlier rows?
            for (int q = lane; q < part * 32; q += 32) seen |= slots[q] == slot;
            if (__any_sync(0xFFFFFFFFu, seen)) continue;
            const bool any = __any_sync(0xFFFFFFFFu, lane < 16 && slots[mine + (lane & 15)] == slot);
            // tiles of eight ranks, set after set
            if (tid < p.sets * (kAdapterMaxRank / 8)) {
                int at = 0, tile = tid;
                for (int set = 0; set < p.sets; ++set) {
                    const AdapterSet &s = p.set[set];
                    const int rt = active(s, slot) ? (s.rank[slot] + 7) / 8 : 0;
                    if (tile >= 0 && tile < rt) {
                        tiles_of[tid].from = reinterpret_cast<const uint4 *>(s.a + slot * s.a_stride) + tile * 32;
                        tiles_of[tid].step = rt * 32;
                        tiles_of[tid].to = s.t_at + 8 * tile;
                    }
                    at += rt;
                    tile -= rt;
                }
                if (tid == 0) all_tiles = at;
            }
            __syncthreads();
            for (int first = 0; first < all_tiles; first += kSumTiles) {
                const int tiles = min(all_tiles - first, kSumTiles);
                float acc[kSumTiles][4];
#pragma unroll
                for (int i = 0; i < kSumTiles; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
                for (int kc = kc0; kc < kc1; kc += BATCH) {
                    const int chunks = min(BATCH, kc1 - kc);
                    __syncthreads();         // what was there has been read
                    for (int i = tid; i < kShrinkRows * 32; i += kThreads) {      // 16 bytes of a row; zeros beyond the rows and K
                        const int r = i >> 5, at = (i & 31) * 16, k = kc * 32 + at / XB;
                        const long long row = base + r;
                        const uint8_t *from = reinterpret_cast<const uint8_t *>(p.x) + (row * p.ldx + k) * XB;
                        uint8_t *to = smem + r * kXLd + at;
                        const int left = row < p.m && at < chunks * 32 * XB ? min(max((p.K - k) * XB, 0), 16) : 0;
                        if (p.x_vec) {
                            if (left == 0) from = reinterpret_cast<const uint8_t *>(p.x);
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(left) : "memory");
                        } else {
#pragma unroll
                            for (int b = 0; b < 16; b += XB) {
                                if (XF32) *reinterpret_cast<uint32_t *>(to + b) = b < left ? *reinterpret_cast<const uint32_t *>(from + b) : 0u;
                                else *reinterpret_cast<uint16_t *>(to + b) = b < left ? *reinterpret_cast<const uint16_t *>(from + b) : (uint16_t)0;
                            }
                        }
                    }
                    for (int i = warp; i < tiles; i += kWarps) {
                        const AdapterTile tile = tiles_of[first + i];
                        for (int c = 0; c < chunks; ++c)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(afrag + ((c * kSumTiles + i) * 32 + lane) * 16)),
                                         "l"(tile.from + (size_t)(kc + c) * tile.step + lane)
                                         : "memory");
                    }
                    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
                    __syncthreads();
                    if (any)
                        for (int c = 0; c < chunks; ++c) {
                            uint32_t f0[PX][4], f1[PX][4];
                            XPiece<XF32> x0, x1;
                            const uint8_t *at = smem + (mine + g) * kXLd + (c * 32 + 8 * t) * XB;
#pragma unroll
                            for (int i = 0; i < (XF32 ? 2 : 1); ++i) {
                                x0.w[i] = *reinterpret_cast<const uint4 *>(at + 16 * i);
                                x1.w[i] = *reinterpret_cast<const uint4 *>(at + 8 * kXLd + 16 * i);
                            }
                            x0.planes(f0);
                            x1.planes(f1);
#pragma unroll
                            for (int i = 0; i < kSumTiles; ++i) {
                                if (i >= tiles) break;
                                multiply_tile<F16, PX>(f0, f1, *reinterpret_cast<const uint4 *>(afrag + ((c * kSumTiles + i) * 32 + lane) * 16), acc[i]);
                            }
                        }
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kSumTiles; ++i) {
                    float *to = sums + (mine + g) * kSumLd + 8 * i + 2 * t;
                    *reinterpret_cast<float2 *>(to) = make_float2(acc[i][0], acc[i][1]);
                    *reinterpret_cast<float2 *>(to + 8 * kSumLd) = make_float2(acc[i][2], acc[i][3]);
                }
                cluster.sync();
                const int rows = kShrinkRows / parts;
                for (int i = tid; i < rows * tiles * 4; i += kThreads) {
                    const int r = part0 * rows + i / (tiles * 4), c = 2 * (i % (tiles * 4));
                    if (slots[r] != slot) continue;
                    float2 o[kCluster], v = make_float2(0.f, 0.f);
#pragma unroll
                    for (int q = 0; q < kCluster; ++q)
                        if (q < parts) o[q] = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(sums, q) + r * kSumLd + c);
#pragma unroll
                    for (int q = 0; q < kCluster; ++q)
                        if (q < parts) v.x += o[q].x, v.y += o[q].y;
                    *reinterpret_cast<float2 *>(p.t + (long long)(base + r) * p.t_ld + tiles_of[first + c / 8].to + c % 8) = v;
                }
                cluster.sync();
            }
            __syncthreads();                 // the tiles' list has been read
        }
}

// y += scale B t: a block takes 64 rows and p.stream_chunks chunks of 32 outputs; four warps side by side in the rows, two in the outputs
constexpr int kStreamRows = 64, kStreamStep = 4;
constexpr size_t kPieces = size_t(kWarps) * 16 * kTileLd * 4;
template <bool F16, bool YF32> __global__ void __launch_bounds__(kThreads, 2) adapters_stream_kernel(const __grid_constant__ AdaptersParams p) {
    constexpr int PT = YF32 ? 3 : 2;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int slots[kStreamRows], row[kStreamRows];
    __shared__ unsigned firsts[2];
    uint4 *frag = reinterpret_cast<uint4 *>(smem + kPieces);
    const AdapterSet &s = p.set[blockIdx.z];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, base = blockIdx.y * kStreamRows;
    const int nc0 = blockIdx.x * p.stream_chunks, nc1 = min(nc0 + p.stream_chunks, s.nchunks);
    if (nc0 >= nc1) return;                  // (another set is wider)
    pdl_launch_dependents();
    pdl_wait();
    if (warp < 2) {
        const int i = warp * 32 + lane;
        int slot = base + i < p.m ? p.rows[base + i] : -1;
        if (!active(s, slot)) slot = -1;
        slots[i] = slot;
        const unsigned first = first_rows(slot, lane);
        if (lane == 0) firsts[warp] = first;
    }
    __syncthreads();
    for (int half = 0; half < 2; ++half)
        for (unsigned left = firsts[half]; left; left &= left - 1) {
            const int slot = slots[half * 32 + __ffs((int)left) - 1];
            if (half == 1) {                 // had its turn among the first rows?
                bool seen = false;
                for (int q = 0; q < 32; ++q) seen |= slots[q] == slot;
                if (seen) continue;
            }
            const int rk = (s.rank[slot] + 15) / 16, ranks = (s.rank[slot] + 7) / 8 * 8;
            if (threadIdx.x < kStreamRows) row[threadIdx.x] = slots[threadIdx.x] == slot ? base + (int)threadIdx.x : -1;
            __syncthreads();
            // t as fragments: [row tile][rank tile][plane][lane]
            for (int i = threadIdx.x; i < 4 * rk * 32; i += kThreads) {
                const int l = i & 31, tile = i >> 5, m = tile / rk, k = tile - m * rk;
                uint32_t w[4][PT];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = row[m * 16 + (l >> 2) + 8 * (e & 1)], c = k * 16 + 2 * (l & 3) + 8 * (e >> 1);
                    float2 v = make_float2(0.f, 0.f);
                    if (r >= 0 && c < ranks) v = *reinterpret_cast<const float2 *>(p.t + (long long)r * p.t_ld + s.t_at + c);
                    split<PT>(v.x, v.y, w[e]);
                }
#pragma unroll
                for (int q = 0; q < PT; ++q) frag[((size_t)tile * PT + q) * 32 + l] = make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
            }
            __syncthreads();
            const int m = warp & 3;
            add_chunks<F16, YF32, kStreamStep>(s, reinterpret_cast<const uint4 *>(s.b + slot * s.b_stride), frag + (size_t)m * rk * PT * 32, rk, s.scale[slot], row + m * 16,
                                               nc0 + (warp >> 2) * kStreamStep, nc1, 2 * kStreamStep, reinterpret_cast<float *>(smem) + warp * 16 * kTileLd, lane);
            __syncthreads();
        }
}

template <typename Kernel> cudaError_t launch(Kernel kern, const AdaptersParams &p, dim3 grid, dim3 cluster, size_t smem, cudaStream_t st) {
    cudaError_t e = configure_smem(reinterpret_cast<const void *>(kern), smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster.x;
    attr[1].val.clusterDim.y = cluster.y;
    attr[1].val.clusterDim.z = cluster.z;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

template <bool F16, bool XF32, bool YF32> cudaError_t run(AdaptersParams p, int sm_count, size_t t_floats, cudaStream_t st) {
    constexpr int PT = YF32 ? 3 : 2;
    if (p.m <= kFewRows) {
        const int clusters = std::min(p.m * p.sets, sm_count * 2 / kCluster);
        return launch(adapters_few_kernel<F16, XF32, YF32>, p, dim3((unsigned)(clusters * kCluster)), dim3(kCluster), few_smem(p.rank_pad, PT), st);
    }
    // blocks that split K: as many as run at a time, of eight chunks each at least
    int parts = kCluster;
    while (parts > 1 && (parts * ((p.m + kShrinkRows - 1) / kShrinkRows) > 2 * sm_count || p.kchunks < 8 * parts)) parts /= 2;
    // A block reads t before its outputs: the more chunks of them, the better, while the SMs have some ten blocks each to share out
    int widest = 0;
    for (int i = 0; i < p.sets; ++i) widest = std::max(widest, p.set[i].nchunks);
    p.stream_chunks = 64;
    while (p.stream_chunks > 8 && (long long)((p.m + kStreamRows - 1) / kStreamRows) * p.sets * ((widest + p.stream_chunks - 1) / p.stream_chunks) < 20ll * sm_count)
        p.stream_chunks /= 2;
    // t of as many rows at a time as there is room for
    const int room = (int)std::min<size_t>(t_floats / (size_t)p.t_ld / kStreamRows * kStreamRows, size_t(32767) * kStreamRows);
    for (int done = 0, all = p.m; done < all; done += room) {
        p.m = std::min(room, all - done);
        cudaError_t e = launch(adapters_shrink_kernel<F16, XF32>, p, dim3((unsigned)((p.m + kShrinkRows - 1) / kShrinkRows), (unsigned)parts), dim3(1, (unsigned)parts),
                               kShrinkSmem, st);
        if (e != cudaSuccess) return e;
        e = launch(adapters_stream_kernel<F16, YF32>, p,
                   dim3((unsigned)((widest + p.stream_chunks - 1) / p.stream_chunks), (unsigned)((p.m + kStreamRows - 1) / kStreamRows), (unsigned)p.sets), dim3(1),
                   kPieces + size_t(4) * (p.rank_pad / 16) * PT * 512, st);
        if (e != cudaSuccess) return e;
        p.rows += p.m;
        p.x = reinterpret_cast<const uint8_t *>(p.x) + (long long)p.m * p.ldx * (XF32 ? 4 : 2);
        for (int i = 0; i < p.sets; ++i) p.set[i].y = reinterpret_cast<uint8_t *>(p.set[i].y) + (long long)p.m * p.set[i].ldy * (YF32 ? 4 : 2);
    }
    return cudaSuccess;
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

cudaError_t adapters_run(const AdaptersParams &p, bool f16, bool x_f32, bool y_f32, int sm_count, size_t t_floats, cudaStream_t st) {
    if (f16) return x_f32 ? (y_f32 ? run<true, true, true>(p, sm_count, t_floats, st) : run<true, true, false>(p, sm_count, t_floats, st))
                          : (y_f32 ? run<true, false, true>(p, sm_count, t_floats, st) : run<true, false, false>(p, sm_count, t_floats, st));
    return x_f32 ? (y_f32 ? run<false, true, true>(p, sm_count, t_floats, st) : run<false, true, false>(p, sm_count, t_floats, st))
                 : (y_f32 ? run<false, false, true>(p, sm_count, t_floats, st) : run<false, false, false>(p, sm_count, t_floats, st));
}

}  // namespace b200q
