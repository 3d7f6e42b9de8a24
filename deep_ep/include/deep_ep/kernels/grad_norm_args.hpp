// Plain-data arguments of the gradient-norm kernels (usable from g++ and nvcc).
#pragma once

#include "../common/math.hpp"

namespace deep_ep::kernels {

enum class GradType : int { kBF16 = 0, kFP16 = 1, kFP32 = 2 };

constexpr int kGradThreads = 256;
constexpr int kGradCtasPerSm = 6;             // 1536 threads with 64 bytes in flight each
constexpr int kGradChunk = 16384;             // elements that are not divided among CTAs
constexpr int kGradCtas = 148 * kGradCtasPerSm;
constexpr int kGradMaxTensors = 1024;         // tensors of one launch: their table travels in the kernel's parameters

// Tensor table, one launch's worth: no copy to the device, nothing to keep alive until the kernel has run. 29 KB of the
// 32 KB that parameters may take; the short form keeps the launch of a few tensors cheap.
template <int kTensors>
struct GradTable {
    const void* in[kTensors];
    void* out[kTensors];                      // scaling only
    int64_t numel[kTensors];
    int first_chunk[kTensors + 1];            // exclusive prefix sum of chunks
    uint8_t in_type[kTensors], out_type[kTensors];
    int num_tensors;
};

struct GradNormArgs {
    double* partial;                          // [kGradCtas] sums of squares, this launch's slots
};

struct GradClipArgs {
    const double* sums;                       // sums of squares to add up
    int num_sums;
    float max_norm;
    float* norm;                              // result (written by CTA 0 of the first launch; may be nullptr)
    int in_place;                             // nothing is written when the factor is 1
};

}  // namespace deep_ep::kernels
