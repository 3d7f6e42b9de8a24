// Plain-data arguments of the adapter kernels (usable from g++ and nvcc).
#pragma once

#include "../common/math.hpp"

namespace deep_ep::kernels {

constexpr int kLoraTileRows = 128;        // token rows of a tile
constexpr int kLoraBlockK = 64;           // 64 bf16 = one 128-byte swizzle row
constexpr int kLoraMaxRank = 128;
constexpr int kLoraMaxCluster = 8;
constexpr int kLoraMaxTileWords = 2048;   // gradients of A and B: bitmap of row tiles ...
constexpr int64_t kLoraMaxGradRows = int64_t(kLoraMaxTileWords) * 32 * kLoraTileRows;        // ... which bounds the rows, 2^23

// Which adapter a row belongs to. An id outside [0, num_adapters) means none.
struct LoraRows {
    const void* idx;                      // int64 or int32 [num_rows]
    int idx64;
    int num_rows, num_adapters, rank;
    int* status;                          // set to 1 if a bounded wait ran out (may be nullptr)
};

// t[row, :] = scaling[e] * (X[row, :] . A_e^T), fp32 [num_rows, rank]; rows without an adapter are not written.
struct LoraShrinkArgs {
    LoraRows rows;
    int k;                                // contraction length
    int mn_major;                         // 0: A_e is [rank, k] (k contiguous); 1: [k, rank] (rank contiguous)
    int chunk, num_chunks;                // adapters per CTA, CTAs per row tile (times the cluster)
    int cluster, ring_bytes;
    const float* scaling;                 // [num_adapters]
    float* t;
    uint8_t* presence;                    // optional [row tiles][num_adapters]: 1 = some row of the tile has the adapter
};

// Y[row, :] = X[row, :] . W^T + t[row, :] . V_e^T, bf16 [num_rows, n].
struct LoraGemmArgs {
    LoraRows rows;
    int k, n;                             // contraction length, columns of Y
    int mn_major;                         // 0: W [n, k], V_e [n, rank]; 1: W [k, n], V_e [rank, n] (the data gradient)
    int cluster;                          // CTAs that share a tile's contraction
    int m_tiles, n_tiles;
    const float* t;                       // fp32 [num_rows, rank], scaled
    const void* v;                        // V, read directly only where it holds infinities or NaN
    void* y;
};

// The same for one row tile and a small low-rank term
struct LoraGemmFewArgs {
    LoraRows rows;
    int k, n, mn_major, cluster;
    int block_n;                          // columns of Y per tile: 64 or 128
    int stage_blocks, num_stages;         // K blocks per stage, stages
    int x_box_rows;                       // rows of X that a load brings: all, up to the next multiple of eight
    const float* t;
    const void* v;
    void* y;
};

// D_e[m, r] = sum over the rows of adapter e of X[row, m] * t[row, r]
struct LoraWgradArgs {
    LoraRows rows;
    int m;                                // columns of X
    int rank_major;                       // 1: the result is [adapters, rank, m], 0: [adapters, m, rank]
    int cluster, num_stages, stage_bytes;
    int m_tiles, row_tiles;
    const float* t;
    const uint8_t* presence;              // [row_tiles][num_adapters]
    void* d;
    int out_fp32, accumulate;             // bf16 (overwrite) or fp32
};

}  // namespace deep_ep::kernels
