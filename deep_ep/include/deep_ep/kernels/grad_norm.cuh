// Global L2 norm over a list of gradient tensors, and clipping by it.
//
// Mathematics: norm = sqrt(sum of g^2 over all tensors), factor = min(1, max_norm / (norm + 1e-6)), g *= factor. Two sweeps
// because the factor needs every element first; both are bound by HBM. The first reads everything once; the second reads
// and writes everything, and when the factor is 1 in place it touches nothing. It walks the chunks from the end, so
// that what the first sweep read last is still in L2 (126 MB).
//
// Sums: the squares of 64 bytes of elements are added in fp32 (at most ten roundings on the way of each), everything above
// that in fp64, whose units would otherwise be the bound for 16-bit gradients. Squares that leave fp32's range (an element
// beyond about 1e18, or all of them below 1e-14) are taken in fp64 instead, so neither huge nor tiny
// gradients lose the norm. Each CTA takes a fixed set of chunks and its sum has a fixed slot: the same bits every time.
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
    if (int(threadIdx.x) < head) acc += square(p[threadIdx.x]);
    if (int(threadIdx.x) < n - tail) acc += square(p[tail + threadIdx.x]);
    const uint4* body = reinterpret_cast<const uint4*>(p + head);
    constexpr int kAhead = 4;
    int i = threadIdx.x;
    for (; i + (kAhead - 1) * kGradThreads < packs; i += kAhead * kGradThreads) {
        uint4 e[kAhead];
        #pragma unroll
        for (int u = 0; u < kAhead; ++u) e[u] = __ldg(body + i + u * kGradThreads);
        const float s = (square_sum<T>(e[0]) + square_sum<T>(e[1])) + (square_sum<T>(e[2]) + square_sum<T>(e[3]));
        if (s > 1e-28f and s < 1e36f) {
            acc += double(s);
        } else {                              // zeros, or a range that fp32 squares do not have (NaN and infinity included)
            #pragma unroll 1
            for (int u = 0; u < kAhead; ++u) acc += square_sum_exact<T>(u == 0 ? e[0] : u == 1 ? e[1] : u == 2 ? e[2] : e[3]);
        }
    }
    for (; i < packs; i += kGradThreads) acc += square_sum_exact<T>(__ldg(body + i));
    return acc;
}

// Eight elements
template <typename T>
struct Eight {
    static constexpr int kUnits = 8 * sizeof(T) / 16;
    uint4 unit[kUnits];
};

template <typename In, typename Out>
EP_DEVICE Eight<Out> scaled(const Eight<In>& in, float factor) {
    float v[8];
    #pragma unroll
    for (int u = 0; u < Eight<In>::kUnits; ++u) {
        const Unpacked<In> e(in.unit[u]);
        #pragma unroll
        for (int j = 0; j < Unpacked<In>::kCount; ++j) v[u * Unpacked<In>::kCount + j] = e.v[j] * factor;
    }
    Eight<Out> out;
    uint32_t w[4 * Eight<Out>::kUnits];
    #pragma unroll
    for (int j = 0; j < 4 * Eight<Out>::kUnits; ++j) {
        if constexpr (sizeof(Out) == 4) {
            w[j] = __float_as_uint(v[j]);
        } else if constexpr (std::is_same_v<Out, __nv_bfloat16>) {
            w[j] = ptx::float2_to_bf16x2(v[2 * j], v[2 * j + 1]);
        } else {
            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    #pragma unroll
    for (int u = 0; u < Eight<Out>::kUnits; ++u) out.unit[u] = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
    return out;
}

template <typename In, typename Out>
__device__ __noinline__ void scale_range(const In* p, Out* q, int n, float factor) {
    // first element from which both sides lie on 16-byte boundaries; none: element by element
    int head = 0;
    while (head < 8 and (((reinterpret_cast<uintptr_t>(p) + head * sizeof(In)) | (reinterpret_cast<uintptr_t>(q) + head * sizeof(Out))) & 15)) ++head;
    if (head == 8) {
        for (int i = threadIdx.x; i < n; i += kGradThreads) q[i] = from_float<Out>(to_float(p[i]) * factor);
        return;
    }
    head = min(head, n);
    const int eights = (n - head) / 8, tail = head + eights * 8;
    if (int(threadIdx.x) < head) q[threadIdx.x] = from_float<Out>(to_float(p[threadIdx.x]) * factor);
    if (int(threadIdx.x) < n - tail) q[tail + threadIdx.x] = from_float<Out>(to_float(p[tail + threadIdx.x]) * factor);
    const uint4* src = reinterpret_cast<const uint4*>(p + head);
    uint4* dst = reinterpret_cast<uint4*>(q + head);
    constexpr int kAhead = 4 / Eight<In>::kUnits;             // 64 bytes a thread in flight
    int i = threadIdx.x;
    for (; i < eights; i += kAhead * kGradThreads) {
        Eight<In> e[kAhead];
        #pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            #pragma unroll
            for (int w = 0; w < Eight<In>::kUnits; ++w)
                if (i + u * kGradThreads < eights) e[u].unit[w] = src[(i + u * kGradThreads) * Eight<In>::kUnits + w];
        }
        #pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i + u * kGradThreads >= eights) break;
            const Eight<Out> o = scaled<In, Out>(e[u], factor);
            #pragma unroll
            for (int w = 0; w < Eight<Out>::kUnits; ++w) dst[(i + u * kGradThreads) * Eight<Out>::kUnits + w] = o.unit[w];
        }
    }
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
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        const int64_t begin = int64_t(chunk - t.first_chunk[i]) * kGradChunk;
        const int n = int(min(int64_t(kGradChunk), t.numel[i] - begin));
        switch (static_cast<GradType>(t.in_type[i])) {
            case GradType::kBF16: acc += sum_range(static_cast<const __nv_bfloat16*>(t.in[i]) + begin, n); break;
            case GradType::kFP16: acc += sum_range(static_cast<const __half*>(t.in[i]) + begin, n); break;
            case GradType::kFP32: acc += sum_range(static_cast<const float*>(t.in[i]) + begin, n); break;
        }
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
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int chunk = chunks - 1 - c;
        const int i = tensor_of(t, chunk);
        const int64_t begin = int64_t(chunk - t.first_chunk[i]) * kGradChunk;
        const int n = int(min(int64_t(kGradChunk), t.numel[i] - begin));
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
