// What the C ABI layer and the kernels of low-rank adapters (adapters.cu) share.
#pragma once

#include "common.cuh"

namespace b200q {

constexpr int kAdapterMaxRank = 256, kAdapterMaxSets = 4;
constexpr size_t kAdapterTFloats = size_t(2) << 20;      // a context's room for t: 2048 rows of 1024 ranks

// Fragments of an adapter, 16 bytes a lane (lane 4 g + t):
//   A  [chunk of 32 of K][rank tile of 8][lane]: rank g of the tile, K 8 t .. 8 t + 7 of the chunk
//   B  [chunk of 32 of N][rank tile of 16][2][lane]: the B operands of two column tiles of mma.m16n8k16; column g of tile v is output
//      8 (g / 2) + 2 v + g % 2 of the chunk, so a lane's results of the four tiles are eight neighbouring outputs
inline int64_t adapter_a_bytes(int64_t rank, int64_t K) { return (K + 31) / 32 * ((rank + 7) / 8) * 512; }
inline int64_t adapter_b_bytes(int64_t rank, int64_t n) { return (n + 31) / 32 * ((rank + 15) / 16) * 1024; }

struct AdapterSet {
    const uint8_t *a, *b;            // slots' fragments
    long long a_stride, b_stride;    // bytes of a slot
    const int *rank;                 // [slot], 0 = nothing loaded
    const float *scale;              // [slot]
    int slots, n, nchunks;
    void *y;
    long long ldy;
    int y_vec;                       // rows of y are 16-byte aligned
    int t_at;                        // more rows: where the set's ranks begin in a row of t
};

struct AdaptersParams {
    AdapterSet set[kAdapterMaxSets];
    int sets;
    const void *x;
    long long ldx;
    int x_vec;
    int K, kchunks;
    const int *rows;                 // [m]: every row's slot
    int m;
    int *status;
    int most_copies;                 // few rows: clusters that may share the outputs of an item
    int rank_pad;                    // largest rank of the sets, in multiples of 16
    // more rows: t = A x on its way from one launch to the next, [row][t_ld]
    float *t;
    int t_ld;
    int stream_chunks;               // chunks of 32 outputs of a block
};

cudaError_t adapter_pack(const void *a, const void *b, uint8_t *pa, uint8_t *pb, int rank, int K, int n, cudaStream_t st);
// t_floats: room at p.t
cudaError_t adapters_run(const AdaptersParams &p, bool f16, bool x_f32, bool y_f32, int sm_count, size_t t_floats, cudaStream_t st);

}  // namespace b200q
