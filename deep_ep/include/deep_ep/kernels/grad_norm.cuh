// Global L2 norm over a list of gradient tensors, and clipping by it.
//
// Mathematics: norm = sqrt(sum of g^2 over all tensors), factor = min(1, max_norm / (norm + 1e-6)), g *= factor. Two sweeps
// because the factor needs every element first; both are bound by HBM. The first reads everything once; the second reads
// and writes everything, and when the factor is 1 in place it touches nothing. It walks from the end to the beginning, so
// that what the first sweep read last is still in L2 (126 MB).
//
// Sums: the squares of 64 bytes of elements are added in fp32 (at most ten roundings on the way of each), everything above
// that in fp64, whose units would otherwise be the bound for 16-bit gradients. Squares that leave fp32's range (an element
// beyond about 1e18, or all of them below 1e-14) are taken in fp64 instead, so neither huge nor tiny
// gradients lose the norm. Each CTA takes a fixed range of chunks and its sum has a fixed slot: the same bits every time.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "../device/ptx.cuh"
#include "grad_norm_args.hpp"

namespace deep_ep::kernels {

namespace grad_detail {

EP_DEVICE float to_float(float v) { return v; }
EP_DEVICE float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
EP_DEVICE float to_float(__half v) { return __half2float(v); }
template <typename T> EP_DEVICE T from_float(float v);
template <> EP_DEVICE float from_float<float>(float v) { return v; }
template <> EP_DEVICE __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> EP_DEVICE __half from_float<__half>(float v) { return __float2half_rn(v); }

// The elements of 16 bytes as floats
template <typename T>
struct Unpacked {
    static constexpr int kCount = 16 / sizeof(T);
    float v[kCount];
    EP_DEVICE explicit Unpacked(const uint4& raw) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
            } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            }
        }
    }
};

template <typename T>
EP_DEVICE float square_sum(const uint4& raw) {
    const Unpacked<T> e(raw);
    float s = 0.0f;
    #pragma unroll
    for (int i = 0; i < Unpacked<T>::kCount; ++i) s = fmaf(e.v[i], e.v[i], s);
    return s;
}
template <typename T>
EP_DEVICE double square_sum_exact(const uint4& raw) {
    const Unpacked<T> e(raw);
    double d = 0.0;
    #pragma unroll
    for (int i = 0; i < Unpacked<T>::kCount; ++i) d += double(e.v[i]) * double(e.v[i]);
    return d;
}
template <typename T>
EP_DEVICE double square(T x) {
    const double v = double(to_float(x));
    return v * v;
}

// Sum of squares of `n` elements by the CTA's threads (each thread's share), 64 bytes a thread in flight
template <typename T>
__device__ __noinline__ double sum_range(const T* p, int n) {
    double acc = 0.0;
    const int head = min(n, int((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / int(sizeof(T)));
    const int packs = (n - head) / Unpacked<T>::kCount, tail = head + packs * Unpacked<T>::kCount;
    const int ends = head + n - tail, end = int(threadIdx.x) < head ? int(threadIdx.x) : tail + int(threadIdx.x) - head;     // what no pack holds
    if (int(threadIdx.x) < ends) acc += square(p[end]);
    const uint4* body = reinterpret_cast<const uint4*>(p + head);
    constexpr int kAhead = 4;
    for (int i = threadIdx.x; i < packs; i += kAhead * kGradThreads) {
        uint4 e[kAhead];
        #pragma unroll
        for (int u = 0; u < kAhead; ++u) e[u] = __ldg(body + min(i + u * kGradThreads, packs - 1));     // (see scale_range)
        #pragma unroll
        for (int u = 1; u < kAhead; ++u)
            if (i + u * kGradThreads >= packs) e[u] = make_uint4(0, 0, 0, 0);
        const float s = (square_sum<T>(e[0]) + square_sum<T>(e[1])) + (square_sum<T>(e[2]) + square_sum<T>(e[3]));
        if (s > 1e-28f and s < 1e36f) {
            acc += double(s);
        } else {                              // zeros, or a range that fp32 squares do not have (NaN and infinity included)
            #pragma unroll 1
            for (int u = 0; u < kAhead; ++u) acc += square_sum_exact<T>(u == 0 ? e[0] : u == 1 ? e[1] : u == 2 ? e[2] : e[3]);
        }
    }
    return acc;
}

// `kBytes` of a tensor
template <int kBytes>
using Unit = std::conditional_t<kBytes == 16, uint4, uint2>;

// As many elements as 16 bytes of the wider type hold, so that both sides move in accesses without gaps between the lanes
template <typename In, typename Out>
constexpr int kScaled = 16 / int(sizeof(In) > sizeof(Out) ? sizeof(In) : sizeof(Out));

template <typename T, int kCount>
EP_DEVICE void to_floats(const Unit<kCount * int(sizeof(T))>& raw, float (&v)[kCount]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
    #pragma unroll
    for (int i = 0; i < kCount; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) v[i] = __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else v[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu)));
    }
}
template <typename T, int kCount>
EP_DEVICE Unit<kCount * int(sizeof(T))> from_floats(const float (&v)[kCount]) {
    Unit<kCount * int(sizeof(T))> raw;
    uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
    #pragma unroll
    for (int i = 0; i < kCount; i += sizeof(T) == 4 ? 1 : 2) {
        if constexpr (sizeof(T) == 4) {
            w[i] = __float_as_uint(v[i]);
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            w[i / 2] = ptx::float2_to_bf16x2(v[i], v[i + 1]);
        } else {
            const __half2 h = __floats2half2_rn(v[i], v[i + 1]);
            w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return raw;
}

template <typename In, typename Out>
__device__ __noinline__ void scale_range(const In* p, Out* q, int n, float factor) {
    constexpr int kCount = kScaled<In, Out>, kInBytes = kCount * int(sizeof(In)), kOutBytes = kCount * int(sizeof(Out));
    // First element from which both sides lie on the boundaries of their accesses, the written one on a sector of 32 bytes if
    // there is such an element (tensors of a bucket begin anywhere); none: element by element.
    const auto first = [&](int out_bytes, int most) {
        int h = 0;
        while (h < most and ((reinterpret_cast<uintptr_t>(p + h) % kInBytes) | (reinterpret_cast<uintptr_t>(q + h) % out_bytes))) ++h;
        return h;
    };
    constexpr int kSector = 32 / int(sizeof(Out));
    int head = first(32, kSector);
    if (head == kSector) head = first(kOutBytes, kCount);
    if (head == kCount and first(kOutBytes, kCount) == kCount) {
        for (int i = threadIdx.x; i < n; i += kGradThreads) q[i] = from_float<Out>(to_float(p[i]) * factor);
        return;
    }
    head = min(head, n);
    const int units = (n - head) / kCount, tail = head + units * kCount;
    const auto* src = reinterpret_cast<const Unit<kInBytes>*>(p + head);
    auto* dst = reinterpret_cast<Unit<kOutBytes>*>(q + head);
    const auto scaled = [&](const Unit<kInBytes>& raw) {
        float v[kCount];
        to_floats<In, kCount>(raw, v);
        #pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] *= factor;
        return from_floats<Out, kCount>(v);
    };
    // Eight loads, then eight stores, without conditions in between: with them the loads were not in flight together (in place,
    // fp32: 4.4 TB/s against 6.4). What eight do not fill comes first (its loads repeat the last unit beyond the end, for
    // nothing), then from the end to the beginning: what the sum has read last is still in L2.
    constexpr int kAhead = 8, kStep = kAhead * kGradThreads;
    const int whole = units / kStep * kStep;
    if (whole < units) {
        const int i = whole + int(threadIdx.x);
        Unit<kInBytes> raw[kAhead];
        #pragma unroll
        for (int u = 0; u < kAhead; ++u) raw[u] = src[min(i + u * kGradThreads, units - 1)];
        #pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (i + u * kGradThreads < units) dst[i + u * kGradThreads] = scaled(raw[u]);
    }
    for (int i = whole - kStep + int(threadIdx.x); i >= 0; i -= kStep) {
        Unit<kInBytes> raw[kAhead];
        #pragma unroll
        for (int u = 0; u < kAhead; ++u) raw[u] = src[i + u * kGradThreads];
        #pragma unroll
        for (int u = 0; u < kAhead; ++u) dst[i + u * kGradThreads] = scaled(raw[u]);
    }
    // what no unit holds
    const int ends = head + n - tail, end = int(threadIdx.x) < head ? int(threadIdx.x) : tail + int(threadIdx.x) - head;
    if (int(threadIdx.x) < ends) q[end] = from_float<Out>(to_float(p[end]) * factor);
}

// Sum over the CTA in a fixed order; valid in every thread
EP_DEVICE double block_sum(double v) {
    __shared__ double warp_sums[kGradThreads / 32];
    __shared__ double total;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (threadIdx.x % 32 == 0) warp_sums[threadIdx.x / 32] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int w = 0; w < kGradThreads / 32; ++w) s += warp_sums[w];
        total = s;
    }
    __syncthreads();
    return total;
}

template <int kTensors>
EP_DEVICE int tensor_of(const GradTable<kTensors>& t, int chunk) {
    int lo = 0, hi = t.num_tensors - 1;
    while (lo < hi) {                         // last tensor whose first chunk is not behind `chunk`
        const int mid = (lo + hi + 1) >> 1;
        if (t.first_chunk[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// first chunk of a CTA's share
EP_DEVICE int share_begin(int chunks, unsigned cta, unsigned ctas) { return static_cast<int>(int64_t(chunks) * cta / ctas); }

EP_DEVICE float clip_factor(float norm, float max_norm) {
    const float f = max_norm / (norm + 1e-6f);
    return f > 1.0f ? 1.0f : f;               // NaN stays NaN
}

}  // namespace grad_detail

template <int kTensors>
__global__ void __launch_bounds__(kGradThreads, kGradCtasPerSm) grad_square_sum_kernel(const __grid_constant__ GradTable<kTensors> t, GradNormArgs a) {
    using namespace grad_detail;
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    const int chunks = t.first_chunk[t.num_tensors];
    double acc = 0.0;
    // a CTA takes consecutive chunks, as long pieces of as few tensors as they lie in
    const int first = share_begin(chunks, blockIdx.x, gridDim.x), last = share_begin(chunks, blockIdx.x + 1, gridDim.x);
    for (int chunk = first; chunk < last; ) {
        const int i = tensor_of(t, chunk), until = min(last, t.first_chunk[i + 1]);
        const int64_t begin = int64_t(chunk - t.first_chunk[i]) * kGradChunk;
        const int n = int(min(int64_t(until - chunk) * kGradChunk, t.numel[i] - begin));
        switch (static_cast<GradType>(t.in_type[i])) {
            case GradType::kBF16: acc += sum_range(static_cast<const __nv_bfloat16*>(t.in[i]) + begin, n); break;
            case GradType::kFP16: acc += sum_range(static_cast<const __half*>(t.in[i]) + begin, n); break;
            case GradType::kFP32: acc += sum_range(static_cast<const float*>(t.in[i]) + begin, n); break;
        }
        chunk = until;
    }
    const double sum = block_sum(acc);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
}

// norm alone: one CTA
__global__ void __launch_bounds__(kGradThreads) grad_norm_finish_kernel(const __grid_constant__ GradClipArgs a) {
    using namespace grad_detail;
    cudaGridDependencySynchronize();          // started early: the sums come from the kernel before
    double acc = 0.0;
    for (int i = threadIdx.x; i < a.num_sums; i += kGradThreads) acc += a.sums[i];
    const double sum = block_sum(acc);
    if (threadIdx.x == 0) *a.norm = static_cast<float>(sqrt(sum));
}

template <int kTensors>
__global__ void __launch_bounds__(kGradThreads, 4) grad_clip_kernel(const __grid_constant__ GradTable<kTensors> t,
                                                                    const __grid_constant__ GradClipArgs a) {
    using namespace grad_detail;
    cudaGridDependencySynchronize();
    // every CTA adds up the few hundred sums itself, which costs less than another launch
    double acc = 0.0;
    for (int i = threadIdx.x; i < a.num_sums; i += kGradThreads) acc += a.sums[i];
    const float norm = static_cast<float>(sqrt(block_sum(acc)));
    if (blockIdx.x == 0 and threadIdx.x == 0 and a.norm != nullptr) *a.norm = norm;
    const float factor = clip_factor(norm, a.max_norm);
    if (a.in_place and factor == 1.0f) return;
    const int chunks = t.first_chunk[t.num_tensors];
    const int first = share_begin(chunks, blockIdx.x, gridDim.x), last = share_begin(chunks, blockIdx.x + 1, gridDim.x);
    for (int until = last; until > first; ) {
        const int i = tensor_of(t, until - 1), chunk = max(first, t.first_chunk[i]);
        const int64_t begin = int64_t(chunk - t.first_chunk[i]) * kGradChunk;
        const int n = int(min(int64_t(until - chunk) * kGradChunk, t.numel[i] - begin));
        until = chunk;
        const auto to = [&](auto* in) {
            switch (static_cast<GradType>(t.out_type[i])) {
                case GradType::kBF16: scale_range(in + begin, static_cast<__nv_bfloat16*>(t.out[i]) + begin, n, factor); break;
                case GradType::kFP16: scale_range(in + begin, static_cast<__half*>(t.out[i]) + begin, n, factor); break;
                case GradType::kFP32: scale_range(in + begin, static_cast<float*>(t.out[i]) + begin, n, factor); break;
            }
        };
        switch (static_cast<GradType>(t.in_type[i])) {
            case GradType::kBF16: to(static_cast<const __nv_bfloat16*>(t.in[i])); break;
            case GradType::kFP16: to(static_cast<const __half*>(t.in[i])); break;
            case GradType::kFP32: to(static_cast<const float*>(t.in[i])); break;
        }
    }
}

}  // namespace deep_ep::kernels
