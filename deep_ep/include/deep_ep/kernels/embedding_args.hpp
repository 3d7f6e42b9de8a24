// Plain-data arguments of the embedding kernels (usable from g++ and nvcc).
#pragma once

#include "../common/math.hpp"

namespace deep_ep::kernels {

enum class EmbType : int { kBF16 = 0, kFP16 = 1, kFP32 = 2, kE4M3 = 3 };

// out[t, :] = table[idx[t], :] * scale (e4m3 tables: times the row's fp32 scale of the 128-column block first);
// rows whose index lies outside [0, num_rows) are zeros.
struct EmbLookupArgs {
    const void* table;
    int64_t table_stride;     // elements between rows
    const float* table_sf;    // e4m3 only: [num_rows, hidden / 128], `sf_stride` elements between rows
    int64_t sf_stride;
    const void* idx;          // int64 or int32 [num_tokens]
    int idx64;
    int64_t num_tokens, num_rows;
    int hidden;
    float scale;
    void* out;                // [num_tokens, hidden]
};

// Stable sort of the token positions by id (least-significant-digit radix sort, `digit_bits` per pass).
struct EmbSortArgs {
    const void* idx;          // int64 or int32 [num_tokens]; ids outside [0, num_rows) become the key `num_rows` (sorted last)
    int idx64;
    int num_tokens, num_rows;
    int digit_bits, num_passes;
    int pass;                 // form of many launches: the pass of this one
    int keys_per_warp;        // form of many launches: contiguous keys of one warp (multiple of 32)
    int *keys[2], *vals[2];   // [num_tokens]; many launches: pass p reads buffer (p + 1) % 2 (pass 0: `idx`) and writes p % 2;
                              // one launch: the result goes to buffer 0
    int* hist;                // form of many launches: [num_ctas][2^digit_bits] counts of this pass
    uint32_t* touched;        // optional bitmap over the rows (bit set = the row receives a gradient)
    int* num_crossing;        // set to 0 for the kernels that follow
};

constexpr int kEmbRankKeys = 8192;            // batches up to this size are ranked by counting (see embedding_rank_kernel)
constexpr int kEmbRankThreads = 1024;
constexpr int kEmbSortThreads = 256;          // form of many launches: eight warps
constexpr int kEmbClusterThreads = 1024;      // form of one launch: a cluster of up to eight CTAs ...
constexpr int kEmbClusterMaxRounds = 8;       // ... with up to this many keys per thread
constexpr int kEmbClusterDigitBits = 9;
constexpr int kEmbMaxDigitBits = 10;

// Sum of the gradient rows of every id over the sorted order, in two steps: chunks of `chunk` sorted positions are reduced
// independently; runs of one id that cross a chunk border leave fp32 partial sums that a second kernel adds in order.
struct EmbGradArgs {
    const void* dy;           // [num_tokens, hidden], `dy_stride` elements between rows
    int64_t dy_stride;
    const int *ids, *order;   // sorted ids (num_rows = none) and the positions they came from
    int num_tokens, num_rows, hidden, chunk, num_chunks;
    float scale;
    float* partial;           // [num_chunks][2][hidden]: the piece of a run that began in an earlier chunk, the piece of one that goes on
    void* out;                // [num_rows, hidden], `out_stride` elements between rows
    int64_t out_stride;
    int accumulate;           // fp32 `out`: add to its contents; otherwise overwrite, rows without a token with zeros
    const uint32_t* touched;  // overwrite: rows without a set bit are written as zeros
    int *num_crossing, *crossing;   // list of the chunks in which a run begins that goes on in the next
};

}  // namespace deep_ep::kernels
