// Embedding lookup with scaling and its gradient (sums over the tokens of an id, in the order of a stable sort).
//
// Mathematics: out[t] = s * table[idx[t]] and dtable[v] = s * sum of dy[t] over the t with idx[t] = v. Both move data and
// compute next to nothing, so both are bound by HBM: the lookup by 2 x tokens x hidden elements, the gradient by reading
// dy once and writing the table's gradient once. Values are scaled, summed and kept in fp32 and rounded once, to the
// type of the result.
//
// The gradient needs no atomics on values: token positions are sorted by id (stable, so the order of the summands is the
// order of the tokens whatever the launch looks like), runs of one id are summed by warps that own a column slice, and
// runs longer than a chunk of sorted positions are joined from fp32 pieces in a fixed order. Two calls with the same
// inputs give the same bits.
#pragma once

#include <cuda_fp16.h>

#include "../device/ptx.cuh"
#include "embedding_args.hpp"

namespace deep_ep::kernels {

namespace emb_detail {

template <int kBytes> struct RawOf;
template <> struct RawOf<1> { using type = uint8_t; };
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };

EP_DEVICE float to_float(float v) { return v; }
EP_DEVICE float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
EP_DEVICE float to_float(__half v) { return __half2float(v); }
EP_DEVICE float to_float(__nv_fp8_e4m3 v) { return static_cast<float>(v); }
template <typename T> EP_DEVICE T from_float(float v);
template <> EP_DEVICE float from_float<float>(float v) { return v; }
template <> EP_DEVICE __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> EP_DEVICE __half from_float<__half>(float v) { return __float2half_rn(v); }

// `kElems` consecutive elements that move as one access of up to 16 bytes (more than that: several of 16)
template <typename T, int kElems>
struct alignas(kElems * sizeof(T) < 16 ? kElems * sizeof(T) : 16) Pack {
    T v[kElems];
};
template <typename T, int kElems>
EP_DEVICE Pack<T, kElems> load_pack(const T* p) {
    using Raw = typename RawOf<(kElems * sizeof(T) < 16 ? kElems * sizeof(T) : 16)>::type;
    constexpr int kParts = kElems * sizeof(T) / sizeof(Raw);
    Pack<T, kElems> out;
    #pragma unroll
    for (int i = 0; i < kParts; ++i) reinterpret_cast<Raw*>(&out)[i] = __ldg(reinterpret_cast<const Raw*>(p) + i);
    return out;
}
template <typename T, int kElems>
EP_DEVICE void store_pack(T* p, const Pack<T, kElems>& in) {
    using Raw = typename RawOf<(kElems * sizeof(T) < 16 ? kElems * sizeof(T) : 16)>::type;
    constexpr int kParts = kElems * sizeof(T) / sizeof(Raw);
    #pragma unroll
    for (int i = 0; i < kParts; ++i) reinterpret_cast<Raw*>(p)[i] = reinterpret_cast<const Raw*>(&in)[i];
}

EP_DEVICE int64_t load_id(const void* idx, int idx64, int64_t i) {
    return idx64 ? reinterpret_cast<const int64_t*>(idx)[i] : reinterpret_cast<const int*>(idx)[i];
}

}  // namespace emb_detail

// One warp per (token, slice of 32 * kElems * kUnroll columns). A warp keeps kUnroll accesses of up to 16 bytes per lane in
// flight: four for large calls, where the 64 resident warps of an SM then cover the latency of HBM; one for small calls,
// which spreads a single row over more SMs.
template <typename In, typename Out, int kElems, int kUnroll>
__global__ void __launch_bounds__(256) embedding_lookup_kernel(const __grid_constant__ EmbLookupArgs a) {
    using namespace emb_detail;
    const int lane = ptx::lane_id();
    const unsigned packs = unsigned(a.hidden) / kElems, slices = math::ceil_div(packs, 32u * kUnroll);
    const unsigned item = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const unsigned token = item / slices, slice = item - token * slices;
    if (token >= a.num_tokens) return;
    const int64_t id = load_id(a.idx, a.idx64, token);
    const bool valid = static_cast<uint64_t>(id) < static_cast<uint64_t>(a.num_rows);
    Out* out = reinterpret_cast<Out*>(a.out) + int64_t(token) * a.hidden;
    const In* row = reinterpret_cast<const In*>(a.table) + (valid ? id : 0) * a.table_stride;
    Pack<In, kElems> in[kUnroll];
    float sf[kUnroll];
    #pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const unsigned p = (slice * kUnroll + u) * 32 + lane;
        sf[u] = 1.0f;
        if (valid and p < packs) {
            in[u] = load_pack<In, kElems>(row + int64_t(p) * kElems);
            if constexpr (sizeof(In) == 1) sf[u] = __ldg(a.table_sf + id * a.sf_stride + p * kElems / 128);
        }
    }
    #pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const unsigned p = (slice * kUnroll + u) * 32 + lane;
        if (p >= packs) continue;
        Pack<Out, kElems> o;
        #pragma unroll
        for (int j = 0; j < kElems; ++j) {
            float v = 0.0f;
            if (valid) v = to_float(in[u].v[j]);
            if constexpr (sizeof(In) == 1) v *= sf[u];
            o.v[j] = from_float<Out>(valid ? v * a.scale : 0.0f);
        }
        store_pack<Out, kElems>(out + int64_t(p) * kElems, o);
    }
}

// ---------------------------------------------------------------------------------------- stable sort by id
namespace emb_detail {

// Key of position i in pass `pass`: the id itself in the first pass (ids outside the table become `num_rows`), the previous
// pass's output afterwards.
EP_DEVICE int sort_key(const EmbSortArgs& a, int pass, int i) {
    if (pass > 0) return a.keys[(pass + 1) & 1][i];
    const int64_t id = load_id(a.idx, a.idx64, i);
    return static_cast<uint64_t>(id) < static_cast<uint64_t>(a.num_rows) ? static_cast<int>(id) : a.num_rows;
}

// Counts of this warp's keys per digit, in `counters` (zeroed by the caller). One lane per distinct digit of a group of 32
// adds the group's count, so that no two lanes touch a counter at once.
EP_DEVICE void sort_count(const EmbSortArgs& a, int pass, int* counters, int begin, int end, int lane) {
    const int mask_bits = (1 << a.digit_bits) - 1, shift = pass * a.digit_bits;
    for (int base = begin; base < end; base += 32) {
        const bool active = base + lane < end;
        const int digit = active ? (sort_key(a, pass, base + lane) >> shift) & mask_bits : mask_bits + 1;
        const unsigned peers = __match_any_sync(0xffffffffu, digit);
        if (active and (peers & ptx::lanemask_lt()) == 0) counters[digit] += __popc(peers);
        __syncwarp();
    }
}

// Writes this warp's keys to their places: `counters[digit]` is the place of the warp's next key with that digit.
EP_DEVICE void sort_scatter(const EmbSortArgs& a, int pass, int* counters, int begin, int end, int lane) {
    const int mask_bits = (1 << a.digit_bits) - 1, shift = pass * a.digit_bits;
    int* out_keys = a.keys[pass & 1];
    int* out_vals = a.vals[pass & 1];
    for (int base = begin; base < end; base += 32) {
        const int i = base + lane;
        const bool active = i < end;
        const int key = active ? sort_key(a, pass, i) : 0;
        const int digit = active ? (key >> shift) & mask_bits : mask_bits + 1;
        const unsigned peers = __match_any_sync(0xffffffffu, digit);
        if (active) {
            const int place = counters[digit] + __popc(peers & ptx::lanemask_lt());
            out_keys[place] = key;
            out_vals[place] = pass > 0 ? a.vals[(pass + 1) & 1][i] : i;
            if (pass == 0 and a.touched != nullptr and key < a.num_rows) atomicOr(a.touched + (key >> 5), 1u << (key & 31));
        }
        __syncwarp();
        if (active and (peers & ptx::lanemask_lt()) == 0) counters[digit] += __popc(peers);
        __syncwarp();
    }
}

// Exclusive prefix sum over `bins` values in shared memory by one CTA of kThreads threads (bins <= kThreads * 4).
template <int kThreads>
EP_DEVICE void block_exclusive_scan(int* values, int bins, int* warp_sums) {
    constexpr int kPer = math::ceil_div(1 << kEmbMaxDigitBits, kThreads);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int local[kPer], sum = 0;
    #pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int b = threadIdx.x * kPer + j;
        local[j] = b < bins ? values[b] : 0;
        sum += local[j];
    }
    int incl = sum;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const int v = lane < kThreads / 32 ? warp_sums[lane] : 0;
        int s = v;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        if (lane < kThreads / 32) warp_sums[lane] = s - v;
    }
    __syncthreads();
    int run = warp_sums[warp] + incl - sum;
    #pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int b = threadIdx.x * kPer + j;
        if (b < bins) values[b] = run;
        run += local[j];
    }
    __syncthreads();
}

// counters[w][b] -> exclusive prefix over the warps, totals[b] = sum over the warps
template <int kWarps>
EP_DEVICE void prefix_over_warps(int* counters, int* totals, int bins) {
    for (int b = threadIdx.x; b < bins; b += kWarps * 32) {
        int run = 0;
        for (int w = 0; w < kWarps; ++w) {
            const int c = counters[w * bins + b];
            counters[w * bins + b] = run;
            run += c;
        }
        totals[b] = run;
    }
    __syncthreads();
}

}  // namespace emb_detail

// All passes in one CTA: no launch gaps between the passes. For the batches whose keys one CTA ranks faster than the four
// launches of the form below take.
__global__ void __launch_bounds__(kEmbSortSoloThreads) embedding_sort_solo_kernel(const __grid_constant__ EmbSortArgs a) {
    using namespace emb_detail;
    constexpr int kWarps = kEmbSortSoloThreads / 32;
    extern __shared__ int sort_smem[];                 // counters [kWarps][bins], totals [bins], warp sums [32]
    const int bins = 1 << a.digit_bits, lane = ptx::lane_id(), warp = threadIdx.x / 32;
    int *totals = sort_smem + kWarps * bins, *warp_sums = totals + bins;
    int* mine = sort_smem + warp * bins;
    const int begin = min(warp * a.keys_per_warp, a.num_tokens), end = min(begin + a.keys_per_warp, a.num_tokens);
    if (a.touched != nullptr)
        for (int i = threadIdx.x; i < (a.num_rows + 31) / 32; i += kEmbSortSoloThreads) a.touched[i] = 0;
    for (int pass = 0; pass < a.num_passes; ++pass) {
        for (int i = threadIdx.x; i < kWarps * bins; i += kEmbSortSoloThreads) sort_smem[i] = 0;
        __syncthreads();
        sort_count(a, pass, mine, begin, end, lane);
        __syncthreads();
        prefix_over_warps<kWarps>(sort_smem, totals, bins);
        block_exclusive_scan<kEmbSortSoloThreads>(totals, bins, warp_sums);
        for (int i = threadIdx.x; i < kWarps * bins; i += kEmbSortSoloThreads) sort_smem[i] += totals[i % bins];
        __syncthreads();
        sort_scatter(a, pass, mine, begin, end, lane);
        __syncthreads();
    }
}

// The same over many CTAs, two launches per pass: counts per CTA, then the scatter (which adds up the counts of the smaller
// digits and of the CTAs before it).
__global__ void __launch_bounds__(kEmbSortThreads) embedding_sort_count_kernel(const __grid_constant__ EmbSortArgs a) {
    using namespace emb_detail;
    constexpr int kWarps = kEmbSortThreads / 32;
    extern __shared__ int sort_smem[];
    const int bins = 1 << a.digit_bits, lane = ptx::lane_id(), warp = threadIdx.x / 32;
    int* totals = sort_smem + kWarps * bins;
    const int64_t first = (int64_t(blockIdx.x) * kWarps + warp) * a.keys_per_warp;
    const int begin = int(min(first, int64_t(a.num_tokens))), end = int(min(first + a.keys_per_warp, int64_t(a.num_tokens)));
    for (int i = threadIdx.x; i < kWarps * bins; i += kEmbSortThreads) sort_smem[i] = 0;
    if (a.pass == 0 and a.touched != nullptr)
        for (int i = blockIdx.x * kEmbSortThreads + threadIdx.x; i < (a.num_rows + 31) / 32; i += gridDim.x * kEmbSortThreads)
            a.touched[i] = 0;
    __syncthreads();
    sort_count(a, a.pass, sort_smem + warp * bins, begin, end, lane);
    __syncthreads();
    prefix_over_warps<kWarps>(sort_smem, totals, bins);
    for (int b = threadIdx.x; b < bins; b += kEmbSortThreads) a.hist[int64_t(blockIdx.x) * bins + b] = totals[b];
}

__global__ void __launch_bounds__(kEmbSortThreads) embedding_sort_scatter_kernel(const __grid_constant__ EmbSortArgs a) {
    using namespace emb_detail;
    constexpr int kWarps = kEmbSortThreads / 32;
    extern __shared__ int sort_smem[];
    const int bins = 1 << a.digit_bits, lane = ptx::lane_id(), warp = threadIdx.x / 32;
    int *totals = sort_smem + kWarps * bins, *before = totals + bins, *warp_sums = before + bins;
    const int64_t first = (int64_t(blockIdx.x) * kWarps + warp) * a.keys_per_warp;
    const int begin = int(min(first, int64_t(a.num_tokens))), end = int(min(first + a.keys_per_warp, int64_t(a.num_tokens)));
    for (int i = threadIdx.x; i < kWarps * bins; i += kEmbSortThreads) sort_smem[i] = 0;
    __syncthreads();
    sort_count(a, a.pass, sort_smem + warp * bins, begin, end, lane);
    __syncthreads();
    prefix_over_warps<kWarps>(sort_smem, totals, bins);
    for (int b = threadIdx.x; b < bins; b += kEmbSortThreads) {
        int all = 0, earlier = 0;
        #pragma unroll 8
        for (int c = 0; c < int(gridDim.x); ++c) {
            const int v = a.hist[int64_t(c) * bins + b];
            all += v;
            earlier += c < int(blockIdx.x) ? v : 0;
        }
        totals[b] = all, before[b] = earlier;
    }
    __syncthreads();
    block_exclusive_scan<kEmbSortThreads>(totals, bins, warp_sums);
    for (int i = threadIdx.x; i < kWarps * bins; i += kEmbSortThreads) sort_smem[i] += totals[i % bins] + before[i % bins];
    __syncthreads();
    sort_scatter(a, a.pass, sort_smem + warp * bins, begin, end, lane);
}

// ---------------------------------------------------------------------------------------- gradient
namespace emb_detail {

template <typename Out, int kElems>
EP_DEVICE void write_sum(const EmbGradArgs& a, int id, int column, const float (&acc)[kElems]) {
    Out* out = reinterpret_cast<Out*>(a.out) + int64_t(id) * a.out_stride + column;
    Pack<Out, kElems> o;
    if constexpr (sizeof(Out) == 4) {
        if (a.accumulate) {
            o = *reinterpret_cast<const Pack<Out, kElems>*>(out);
            #pragma unroll
            for (int j = 0; j < kElems; ++j) o.v[j] += a.scale * acc[j];
            store_pack<Out, kElems>(out, o);
            return;
        }
    }
    #pragma unroll
    for (int j = 0; j < kElems; ++j) o.v[j] = from_float<Out>(a.scale * acc[j]);
    store_pack<Out, kElems>(out, o);
}

template <int kElems>
EP_DEVICE void write_partial(float* p, const float (&acc)[kElems]) {
    Pack<float, kElems> o;
    #pragma unroll
    for (int j = 0; j < kElems; ++j) o.v[j] = acc[j];
    store_pack<float, kElems>(p, o);
}

}  // namespace emb_detail

// One warp per (chunk of sorted positions, slice of 32 * kElems columns): the rows of a run are added in registers, kAhead
// loads in flight. Further warps write the zero rows of a dense gradient, whose bytes are most of the work when the table is
// much larger than the batch.
template <typename In, typename Out, int kElems>
__global__ void __launch_bounds__(256) embedding_grad_kernel(const __grid_constant__ EmbGradArgs a) {
    using namespace emb_detail;
    constexpr int kAhead = 8;
    const int lane = ptx::lane_id();
    const unsigned slices = math::ceil_div(unsigned(a.hidden), 32u * kElems);
    const int64_t item = int64_t(blockIdx.x) * 8 + threadIdx.x / 32;
    const int64_t sum_items = int64_t(a.num_chunks) * slices;
    if (item >= sum_items) {
        // ---- rows without a token
        const int64_t row = item - sum_items;
        if (a.touched == nullptr or row >= a.num_rows or ((a.touched[row >> 5] >> (row & 31)) & 1u)) return;
        Pack<Out, kElems> zero;
        #pragma unroll
        for (int j = 0; j < kElems; ++j) zero.v[j] = from_float<Out>(0.0f);
        for (int c = lane * kElems; c < a.hidden; c += 32 * kElems)
            store_pack<Out, kElems>(reinterpret_cast<Out*>(a.out) + row * a.out_stride + c, zero);
        return;
    }
    const int chunk = int(unsigned(item) / slices), slice = int(unsigned(item) - unsigned(chunk) * slices);
    const int column = (slice * 32 + lane) * kElems;
    const bool mine = column < a.hidden;
    const int begin = chunk * a.chunk, end = min(begin + a.chunk, a.num_tokens);
    int run = a.ids[begin];
    bool from_before = begin > 0 and a.ids[begin - 1] == run;
    const int next = end < a.num_tokens ? a.ids[end] : a.num_rows;
    float acc[kElems];
    #pragma unroll
    for (int j = 0; j < kElems; ++j) acc[j] = 0.0f;

    auto flush = [&](bool goes_on) {
        if (run >= a.num_rows or not mine) return;
        if (from_before) write_partial<kElems>(a.partial + (int64_t(chunk) * 2) * a.hidden + column, acc);
        else if (goes_on) write_partial<kElems>(a.partial + (int64_t(chunk) * 2 + 1) * a.hidden + column, acc);
        else write_sum<Out, kElems>(a, run, column, acc);
    };

    for (int base = begin; base < end; base += 32) {
        const int count = min(32, end - base);
        const int my_id = lane < count ? a.ids[base + lane] : a.num_rows;
        const int my_row = lane < count ? a.order[base + lane] : 0;
        if (__shfl_sync(0xffffffffu, my_id, 0) >= a.num_rows and run >= a.num_rows) return;    // only masked positions follow
        for (int j0 = 0; j0 < count; j0 += kAhead) {
            Pack<In, kElems> in[kAhead];
            #pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int id = __shfl_sync(0xffffffffu, my_id, j0 + u), row = __shfl_sync(0xffffffffu, my_row, j0 + u);
                if (id < a.num_rows and mine)
                    in[u] = load_pack<In, kElems>(reinterpret_cast<const In*>(a.dy) + int64_t(row) * a.dy_stride + column);
            }
            #pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int id = __shfl_sync(0xffffffffu, my_id, j0 + u);
                if (j0 + u >= count) break;
                if (id != run) {
                    flush(false);
                    run = id, from_before = false;
                    #pragma unroll
                    for (int j = 0; j < kElems; ++j) acc[j] = 0.0f;
                }
                if (id < a.num_rows and mine) {
                    #pragma unroll
                    for (int j = 0; j < kElems; ++j) acc[j] += to_float(in[u].v[j]);
                }
            }
        }
    }
    flush(end < a.num_tokens and next == run);
}

// Runs that cross chunk borders. The CTA of the chunk in which such a run begins adds its pieces: eight warps take consecutive
// ranges of them, and the eight sums are added in order.
template <typename Out, int kElems>
__global__ void __launch_bounds__(256) embedding_grad_join_kernel(const __grid_constant__ EmbGradArgs a) {
    using namespace emb_detail;
    __shared__ float sums[8][32 * kElems];
    const int lane = ptx::lane_id(), warp = threadIdx.x / 32, chunk = blockIdx.x;
    const int begin = chunk * a.chunk, end = min(begin + a.chunk, a.num_tokens);
    if (end >= a.num_tokens) return;
    const int id = a.ids[end - 1];
    if (id >= a.num_rows or a.ids[end] != id) return;                               // nothing goes on
    if (begin > 0 and a.ids[begin] == id and a.ids[begin - 1] == id) return;        // it began earlier
    // last chunk whose first position still belongs to the run
    int lo = chunk + 1, hi = a.num_chunks - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.ids[int64_t(mid) * a.chunk] == id) lo = mid; else hi = mid - 1;
    }
    const int pieces = lo - chunk;                                                  // pieces in the chunks chunk + 1 .. lo
    const int per_warp = math::ceil_div(pieces, 8);
    const int first = min(warp * per_warp, pieces), last = min(first + per_warp, pieces);
    const int slices = math::ceil_div(a.hidden, 32 * kElems);
    for (int slice = blockIdx.y; slice < slices; slice += gridDim.y) {
        const int column = (slice * 32 + lane) * kElems;
        float acc[kElems];
        #pragma unroll
        for (int j = 0; j < kElems; ++j) acc[j] = 0.0f;
        if (column < a.hidden) {
            if (warp == 0) {
                const auto head = *reinterpret_cast<const Pack<float, kElems>*>(a.partial + (int64_t(chunk) * 2 + 1) * a.hidden + column);
                #pragma unroll
                for (int j = 0; j < kElems; ++j) acc[j] = head.v[j];
            }
            #pragma unroll 4
            for (int i = first; i < last; ++i) {
                const auto p = *reinterpret_cast<const Pack<float, kElems>*>(a.partial + (int64_t(chunk + 1 + i) * 2) * a.hidden + column);
                #pragma unroll
                for (int j = 0; j < kElems; ++j) acc[j] += p.v[j];
            }
        }
        #pragma unroll
        for (int j = 0; j < kElems; ++j) sums[warp][lane * kElems + j] = acc[j];
        __syncthreads();
        if (warp == 0 and column < a.hidden) {
            #pragma unroll
            for (int j = 0; j < kElems; ++j) acc[j] = sums[0][lane * kElems + j];
            for (int w = 1; w < 8; ++w) {
                #pragma unroll
                for (int j = 0; j < kElems; ++j) acc[j] += sums[w][lane * kElems + j];
            }
            write_sum<Out, kElems>(a, id, column, acc);
        }
        __syncthreads();
    }
}

}  // namespace deep_ep::kernels
