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

#include <type_traits>

#include "../device/tcgen05.cuh"
#include "embedding_args.hpp"

namespace deep_ep::kernels {

namespace emb_detail {

// `kElems` consecutive elements as they move: one access of up to 16 bytes, or two of 16. Kept as raw words until they are used
// (elements of 16 bits would otherwise take a register each).
template <typename T, int kElems>
struct Pack {
    static constexpr int kBytes = kElems * int(sizeof(T)), kParts = kBytes > 16 ? kBytes / 16 : 1;
    using Raw = std::conditional_t<kBytes >= 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, uint32_t,
                std::conditional_t<kBytes == 2, uint16_t, uint8_t>>>>;
    Raw raw[kParts];

    EP_DEVICE uint32_t word(int i) const {
        if constexpr (kBytes >= 16) {
            const uint4& u = raw[i / 4];
            return i % 4 == 0 ? u.x : i % 4 == 1 ? u.y : i % 4 == 2 ? u.z : u.w;
        } else if constexpr (kBytes == 8) {
            return i == 0 ? raw[0].x : raw[0].y;
        } else {
            return raw[0];
        }
    }
    EP_DEVICE void set_word(int i, uint32_t w) {
        if constexpr (kBytes >= 16) {
            uint4& u = raw[i / 4];
            (i % 4 == 0 ? u.x : i % 4 == 1 ? u.y : i % 4 == 2 ? u.z : u.w) = w;
        } else if constexpr (kBytes == 8) {
            (i == 0 ? raw[0].x : raw[0].y) = w;
        } else {
            raw[0] = static_cast<Raw>(w);
        }
    }
};

template <typename T, int kElems>
EP_DEVICE Pack<T, kElems> load_pack(const T* p) {           // data that nobody writes during the kernel
    Pack<T, kElems> out;
    #pragma unroll
    for (int i = 0; i < Pack<T, kElems>::kParts; ++i) out.raw[i] = __ldg(reinterpret_cast<const typename Pack<T, kElems>::Raw*>(p) + i);
    return out;
}
template <typename T, int kElems>
EP_DEVICE Pack<T, kElems> load_written_pack(const T* p) {
    Pack<T, kElems> out;
    #pragma unroll
    for (int i = 0; i < Pack<T, kElems>::kParts; ++i) out.raw[i] = reinterpret_cast<const typename Pack<T, kElems>::Raw*>(p)[i];
    return out;
}
template <typename T, int kElems>
EP_DEVICE void store_pack(T* p, const Pack<T, kElems>& in) {
    #pragma unroll
    for (int i = 0; i < Pack<T, kElems>::kParts; ++i) reinterpret_cast<typename Pack<T, kElems>::Raw*>(p)[i] = in.raw[i];
}

template <typename T, int kElems>
EP_DEVICE void unpack(const Pack<T, kElems>& in, float (&out)[kElems]) {
    if constexpr (sizeof(T) == 4) {
        #pragma unroll
        for (int j = 0; j < kElems; ++j) out[j] = __uint_as_float(in.word(j));
    } else if constexpr (sizeof(T) == 2) {
        #pragma unroll
        for (int j = 0; j < kElems; ++j) {
            const uint32_t w = in.word(j / 2);
            if constexpr (std::is_same_v<T, __nv_bfloat16>) out[j] = __uint_as_float(j % 2 ? w & 0xffff0000u : w << 16);
            else out[j] = __half2float(__ushort_as_half(static_cast<unsigned short>(j % 2 ? w >> 16 : w & 0xffffu)));
        }
    } else if constexpr (kElems == 1) {
        out[0] = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(in.word(0)), __NV_E4M3)));
    } else {
        #pragma unroll
        for (int j = 0; j < kElems; j += 2) {               // the hardware converts pairs
            const uint32_t w = in.word(j / 4);
            const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(j % 4 ? w >> 16 : w & 0xffffu), __NV_E4M3)));
            out[j] = f.x, out[j + 1] = f.y;
        }
    }
}
// Rounds to the type
template <typename T, int kElems>
EP_DEVICE Pack<T, kElems> pack(const float (&v)[kElems]) {
    Pack<T, kElems> out;
    if constexpr (sizeof(T) == 4) {
        #pragma unroll
        for (int j = 0; j < kElems; ++j) out.set_word(j, __float_as_uint(v[j]));
    } else {
        #pragma unroll
        for (int j = 0; j < kElems; j += 2) {
            const float next = j + 1 < kElems ? v[j + 1 < kElems ? j + 1 : j] : 0.0f;
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                out.set_word(j / 2, ptx::float2_to_bf16x2(v[j], next));
            } else {
                const __half2 h = __floats2half2_rn(v[j], next);
                out.set_word(j / 2, *reinterpret_cast<const uint32_t*>(&h));
            }
        }
    }
    return out;
}

EP_DEVICE int64_t load_id(const void* idx, int idx64, int64_t i) {
    return idx64 ? reinterpret_cast<const int64_t*>(idx)[i] : reinterpret_cast<const int*>(idx)[i];
}

}  // namespace emb_detail

// One warp per (token, slice of 32 * kElems * kUnroll columns). The side with the wider elements moves 16 bytes per lane and
// access (8-bit entries are therefore read 8 bytes at a time: 16 would leave stores of half sectors). A warp keeps kUnroll
// accesses per lane in flight: four for large calls, where the 64 resident warps of an SM then cover the latency of HBM; one for small calls,
// which spreads a single row over more SMs.
template <typename In, typename Out, int kElems, int kUnroll>
__global__ void __launch_bounds__(256) embedding_lookup_kernel(const __grid_constant__ EmbLookupArgs a) {
    using namespace emb_detail;
    const int lane = ptx::lane_id();
    const unsigned packs = unsigned(a.hidden) / kElems, slices = math::ceil_div(packs, 32u * kUnroll);
    const unsigned item = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const unsigned token = item / slices, slice = item - token * slices;
    cudaGridDependencySynchronize();
    if (token >= a.num_tokens) return;
    const int64_t id = load_id(a.idx, a.idx64, token);
    const bool valid = static_cast<uint64_t>(id) < static_cast<uint64_t>(a.num_rows);
    Out* out = reinterpret_cast<Out*>(a.out) + int64_t(token) * a.hidden;
    const In* row = reinterpret_cast<const In*>(a.table) + (valid ? id : 0) * a.table_stride;
    Pack<In, kElems> in[kUnroll];
    float sf[kUnroll];
    if (valid) {
        // (no condition per load: lanes beyond the row's end repeat its last pack, for nothing)
        #pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const unsigned p = min((slice * kUnroll + u) * 32 + lane, packs - 1);
            in[u] = load_pack<In, kElems>(row + int64_t(p) * kElems);
            sf[u] = 1.0f;
            if constexpr (sizeof(In) == 1) sf[u] = __ldg(a.table_sf + id * a.sf_stride + p * kElems / 128);
        }
    }
    #pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const unsigned p = (slice * kUnroll + u) * 32 + lane;
        if (p >= packs) continue;
        float v[kElems];
        unpack<In, kElems>(in[u], v);
        #pragma unroll
        for (int j = 0; j < kElems; ++j) {
            if constexpr (sizeof(In) == 1) v[j] *= sf[u];
            v[j] = valid ? v[j] * a.scale : 0.0f;
        }
        store_pack<Out, kElems>(out + int64_t(p) * kElems, pack<Out, kElems>(v));
    }
}

// ---------------------------------------------------------------------------------------- stable sort by id
namespace emb_detail {

// (the bitmap is zero before the sort begins)
EP_DEVICE void mark_touched(const EmbSortArgs& a, int key) {
    if (a.touched != nullptr and key < a.num_rows) atomicOr(a.touched + (key >> 5), 1u << (key & 31));
}

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
            if (pass == 0) mark_touched(a, key);
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

// Small batches: the place of a key is the number of keys before it (smaller, or equal and earlier), counted outright. A CTA
// counts for 32 keys, its 32 warps over a part of all keys each. n^2 comparisons are 67 million for 8192 keys, 2 us of this
// GPU, and there is nothing to wait for in between; a radix sort has a chain of barriers per digit. Whole gradient calls of 64
// columns with this kernel | the next one, us: 512 tokens 8.9 | 13.7, 4096 13.7 | 23.3, 8192 21.9 | 25.7.
__global__ void __launch_bounds__(kEmbRankThreads) embedding_rank_kernel(const __grid_constant__ EmbSortArgs a) {
    using namespace emb_detail;
    extern __shared__ int sort_smem[];                 // all keys, padded to a multiple of 32 with the largest number
    __shared__ int counts[32];
    constexpr int kWarps = kEmbRankThreads / 32;
    const int lane = ptx::lane_id(), warp = threadIdx.x / 32, n = a.num_tokens, padded = math::align(n, 32);
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();         // the kernel of the sums may be set up meanwhile
    if (blockIdx.x == 0 and threadIdx.x == 0) *a.num_crossing = 0;
    if (threadIdx.x < 32) counts[threadIdx.x] = 0;
    #pragma unroll 8
    for (int i = threadIdx.x; i < padded; i += kEmbRankThreads) sort_smem[i] = i < n ? sort_key(a, 0, i) : 0x7fffffff;
    __syncthreads();
    const int first = blockIdx.x * 32, mine = first + lane, key = sort_smem[mine];
    const int per_warp = math::align(math::ceil_div(padded, kWarps), 32);
    const int begin = min(warp * per_warp, padded), end = min(begin + per_warp, padded);
    int count = 0;
    // in groups of 32: those before this CTA's count smaller or equal keys, those behind it smaller ones, its own equal ones in
    // lower lanes too
    #pragma unroll 1
    for (int group = begin; group < end; group += 32) {
        const int limit = group < first ? key + 1 : key;
        #pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const int4 k = *reinterpret_cast<const int4*>(sort_smem + group + j);
            count += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
        }
        if (group == first) count += __popc(__match_any_sync(0xffffffffu, key) & ptx::lanemask_lt());
    }
    atomicAdd(&counts[lane], count);
    __syncthreads();
    if (warp == 0 and mine < n) {
        a.keys[0][counts[lane]] = key, a.vals[0][counts[lane]] = mine;
        mark_touched(a, key);
    }
}

// All passes in one launch: up to eight CTAs of a cluster hold the keys in their shared memory. Per pass every warp ranks its
// keys (in registers) per digit, the CTAs exchange their counts, and each key goes straight into the shared memory of the CTA
// that owns its place (the last pass writes to memory). The time is latency (match, barriers), not work, so the keys are
// spread over the cluster even when one CTA could hold them: a warp then has one or two rounds of 32 keys. Whole gradient calls of
// 64 columns with this kernel | the launches per digit below, us: 16384 tokens 26.8 | 49.2, 32768 40.7 | 56.7, 65536 68.7 | 67.8.
template <int kRounds>
__global__ void __launch_bounds__(kEmbClusterThreads, 1) embedding_sort_cluster_kernel(const __grid_constant__ EmbSortArgs a) {
    using namespace emb_detail;
    constexpr int kWarps = kEmbClusterThreads / 32, kKeys = kEmbClusterThreads * kRounds;       // keys of a CTA, a power of two
    extern __shared__ int sort_smem[];
    __shared__ int warp_sums[32];
    const int bins = 1 << a.digit_bits, lane = ptx::lane_id(), warp = threadIdx.x / 32;
    const int rank = int(tc::cluster_ctarank()), ctas = int(gridDim.x);
    int* keys[2] = {sort_smem, sort_smem + kKeys};
    int* vals[2] = {sort_smem + 2 * kKeys, sort_smem + 3 * kKeys};
    int *hist = sort_smem + 4 * kKeys, *base = hist + bins, *totals = base + bins;
    uint16_t* counters = reinterpret_cast<uint16_t*>(totals + bins);                            // [kWarps][bins]
    uint16_t* mine = counters + warp * bins;
    const int count = min(max(a.num_tokens - rank * kKeys, 0), kKeys);                          // this CTA's keys

    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();                  // the kernel of the sums may be set up meanwhile
    if (rank == 0 and threadIdx.x == 0) *a.num_crossing = 0;
    int key[kRounds], val[kRounds];
    #pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const int i = (warp * kRounds + r) * 32 + lane;
        val[r] = rank * kKeys + i;
        key[r] = i < count ? sort_key(a, 0, val[r]) : a.num_rows;
        mark_touched(a, key[r]);
    }
    for (int pass = 0; pass < a.num_passes; ++pass) {
        const int shift = pass * a.digit_bits;
        if (pass > 0) {
            #pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int i = (warp * kRounds + r) * 32 + lane;
                if (i < count) key[r] = keys[pass & 1][i], val[r] = vals[pass & 1][i];
            }
        }
        for (int i = threadIdx.x; i < kWarps * bins / 2; i += kEmbClusterThreads) reinterpret_cast<uint32_t*>(counters)[i] = 0;
        __syncthreads();
        int place[kRounds];                   // among this warp's keys of the same digit
        #pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const bool active = (warp * kRounds + r) * 32 + lane < count;
            const int digit = active ? (key[r] >> shift) & (bins - 1) : bins;
            const unsigned peers = __match_any_sync(0xffffffffu, digit);
            const int before = __popc(peers & ptx::lanemask_lt());
            place[r] = active ? mine[digit] + before : 0;
            __syncwarp();
            if (active and before == 0) mine[digit] += uint16_t(__popc(peers));
            __syncwarp();
        }
        __syncthreads();
        for (int b = threadIdx.x; b < bins; b += kEmbClusterThreads) {
            int run = 0;
            #pragma unroll 8
            for (int w = 0; w < kWarps; ++w) {
                const int c = counters[w * bins + b];
                counters[w * bins + b] = uint16_t(run);
                run += c;
            }
            hist[b] = run;
        }
        tc::cluster_sync();
        for (int b = threadIdx.x; b < bins; b += kEmbClusterThreads) {
            int all = 0, earlier = 0;
            int v[8];
            #pragma unroll
            for (int q = 0; q < 8; ++q)       // all in flight at once
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v[q]) : "r"(tc::map_to_cta(hist + b, min(q, ctas - 1))));
            #pragma unroll
            for (int q = 0; q < 8; ++q) {
                all += q < ctas ? v[q] : 0;
                earlier += q < rank ? v[q] : 0;
            }
            totals[b] = all, base[b] = earlier;
        }
        __syncthreads();
        block_exclusive_scan<kEmbClusterThreads>(totals, bins, warp_sums);
        const bool last = pass + 1 == a.num_passes;
        #pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            if ((warp * kRounds + r) * 32 + lane >= count) continue;
            const int digit = (key[r] >> shift) & (bins - 1);
            const int at = totals[digit] + base[digit] + mine[digit] + place[r];
            if (last) {
                a.keys[0][at] = key[r], a.vals[0][at] = val[r];
            } else {
                const int q = at / kKeys, i = at % kKeys, to = (pass + 1) & 1;
                asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(tc::map_to_cta(keys[to] + i, q)), "r"(key[r]) : "memory");
                asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(tc::map_to_cta(vals[to] + i, q)), "r"(val[r]) : "memory");
            }
        }
        tc::cluster_sync();                   // keys are in place, and nobody still reads a neighbour's counts
    }
}

// Longer inputs: any number of CTAs, two launches per pass (counts per CTA, then the scatter, which adds up the counts of the
// smaller digits and of the CTAs before it), keys in memory.
__global__ void __launch_bounds__(kEmbSortThreads) embedding_sort_count_kernel(const __grid_constant__ EmbSortArgs a) {
    using namespace emb_detail;
    constexpr int kWarps = kEmbSortThreads / 32;
    extern __shared__ int sort_smem[];
    const int bins = 1 << a.digit_bits, lane = ptx::lane_id(), warp = threadIdx.x / 32;
    int* totals = sort_smem + kWarps * bins;
    const int64_t first = (int64_t(blockIdx.x) * kWarps + warp) * a.keys_per_warp;
    const int begin = int(min(first, int64_t(a.num_tokens))), end = int(min(first + a.keys_per_warp, int64_t(a.num_tokens)));
    for (int i = threadIdx.x; i < kWarps * bins; i += kEmbSortThreads) sort_smem[i] = 0;
    if (a.pass == 0 and blockIdx.x == 0 and threadIdx.x == 0) *a.num_crossing = 0;
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
EP_DEVICE void write_sum(Out* out, float scale, const float (&acc)[kElems]) {
    float v[kElems];
    #pragma unroll
    for (int j = 0; j < kElems; ++j) v[j] = scale * acc[j];
    store_pack<Out, kElems>(out, pack<Out, kElems>(v));
}
// The same added to what was there (`old`, read ahead)
template <int kElems>
EP_DEVICE void add_sum(float* out, float scale, const float (&acc)[kElems], const Pack<float, kElems>& old) {
    float v[kElems];
    unpack<float, kElems>(old, v);
    #pragma unroll
    for (int j = 0; j < kElems; ++j) v[j] += scale * acc[j];
    store_pack<float, kElems>(out, pack<float, kElems>(v));
}

}  // namespace emb_detail

// One warp per (chunk of sorted positions, slice of 32 * kElems * kPacks columns): the rows of a run are added in registers,
// kAhead rows in flight. When the sums are added to a buffer, the rows that end in the group of kAhead are read ahead too:
// a read at the end of each run would be a round trip to memory per id. Further warps write the zero rows of a dense gradient,
// whose bytes are most of the work when the table is much larger than the batch; a row each, so that they end together
// (a range of rows per CTA, with the range's ids searched for instead of marked, took a third longer).
template <typename In, typename Out, int kElems, int kPacks, bool kAccumulate>
__global__ void __launch_bounds__(256, 3) embedding_grad_kernel(const __grid_constant__ EmbGradArgs a) {
    using namespace emb_detail;
    constexpr int kAhead = kAccumulate ? 4 : 8;
    const int lane = ptx::lane_id();
    cudaGridDependencySynchronize();                            // the sort is done
    cudaTriggerProgrammaticLaunchCompletion();                  // the join kernel, or whatever comes next, may be set up meanwhile
    const unsigned slices = math::ceil_div(unsigned(a.hidden), 32u * kElems * kPacks);
    const int64_t item = int64_t(blockIdx.x) * 8 + threadIdx.x / 32, sum_items = int64_t(a.num_chunks) * slices;
    if (item >= sum_items) {
        // ---- rows without a token
        const int64_t row = item - sum_items;
        if (a.accumulate or row >= a.num_rows or ((a.touched[row >> 5] >> (row & 31)) & 1u)) return;
        const float nothing[kElems] = {};
        const Pack<Out, kElems> zero = pack<Out, kElems>(nothing);
        for (int c = lane * kElems; c < a.hidden; c += 32 * kElems)
            store_pack<Out, kElems>(reinterpret_cast<Out*>(a.out) + row * a.out_stride + c, zero);
        return;
    }
    const int chunk = int(unsigned(item) / slices), slice = int(unsigned(item) - unsigned(chunk) * slices);
    constexpr int kWidth = 32 * kElems;                         // columns from one pack of a lane to its next
    const int column = slice * (kWidth * kPacks) + lane * kElems;
    bool mine[kPacks];
    #pragma unroll
    for (int p = 0; p < kPacks; ++p) mine[p] = column + p * kWidth < a.hidden;
    const int begin = chunk * a.chunk, end = min(begin + a.chunk, a.num_tokens);
    bool from_before = begin > 0 and a.ids[begin - 1] == a.ids[begin];
    const In* dy = reinterpret_cast<const In*>(a.dy) + column;
    float* partial = a.partial + int64_t(chunk) * 2 * a.hidden + column;
    float acc[kPacks][kElems] = {};

    for (int base = begin; base < end; base += 32) {
        const int count = min(32, end - base);
        const int my_id = lane < count ? a.ids[base + lane] : a.num_rows;
        const int my_row = lane < count ? a.order[base + lane] : 0;
        const int behind = base + count < a.num_tokens ? a.ids[base + count] : a.num_rows;
        // positions with an id (they come first), and those that end a run
        const int valid = __popc(__ballot_sync(0xffffffffu, my_id < a.num_rows));
        int after = __shfl_down_sync(0xffffffffu, my_id, 1);
        if (lane == count - 1) after = behind;
        const unsigned ends = __ballot_sync(0xffffffffu, after != my_id);
        for (int j0 = 0; j0 < valid; j0 += kAhead) {
            Pack<In, kElems> in[kAhead][kPacks];
            Pack<float, kAccumulate ? kElems : 1> old[kAhead][kPacks];
            #pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (j0 + u >= valid) break;
                const In* src = dy + int64_t(__shfl_sync(0xffffffffu, my_row, j0 + u)) * a.dy_stride;
                #pragma unroll
                for (int p = 0; p < kPacks; ++p)
                    if (mine[p]) in[u][p] = load_pack<In, kElems>(src + p * kWidth);
                if constexpr (kAccumulate) {
                    if ((ends >> (j0 + u)) & 1u) {
                        const float* out = reinterpret_cast<const float*>(a.out) + int64_t(__shfl_sync(0xffffffffu, my_id, j0 + u)) * a.out_stride + column;
                        #pragma unroll
                        for (int p = 0; p < kPacks; ++p)
                            if (mine[p]) old[u][p] = load_written_pack<float, kElems>(out + p * kWidth);
                    }
                }
            }
            #pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (j0 + u >= valid) break;
                #pragma unroll
                for (int p = 0; p < kPacks; ++p) {
                    float v[kElems];
                    unpack<In, kElems>(in[u][p], v);
                    #pragma unroll
                    for (int j = 0; j < kElems; ++j) acc[p][j] += v[j];
                }
                const bool run_ends = (ends >> (j0 + u)) & 1u, last = base + j0 + u == end - 1;
                if (not run_ends and not last) continue;
                if (from_before or not run_ends) {
                    // a piece of a run that crosses a chunk border; one that begins here and goes on enters the list for the
                    // join kernel (in whatever order: runs do not meet)
                    #pragma unroll
                    for (int p = 0; p < kPacks; ++p)
                        if (mine[p]) store_pack<float, kElems>(partial + (from_before ? 0 : a.hidden) + p * kWidth, pack<float, kElems>(acc[p]));
                    if (not from_before and slice == 0 and lane == 0) a.crossing[atomicAdd(a.num_crossing, 1)] = chunk;
                } else {
                    Out* out = reinterpret_cast<Out*>(a.out) + int64_t(__shfl_sync(0xffffffffu, my_id, j0 + u)) * a.out_stride + column;
                    #pragma unroll
                    for (int p = 0; p < kPacks; ++p) {
                        if (not mine[p]) continue;
                        if constexpr (kAccumulate) add_sum<kElems>(out + p * kWidth, a.scale, acc[p], old[u][p]);
                        else write_sum<Out, kElems>(out + p * kWidth, a.scale, acc[p]);
                    }
                }
                from_before = false;
                #pragma unroll
                for (int p = 0; p < kPacks; ++p)
                    #pragma unroll
                    for (int j = 0; j < kElems; ++j) acc[p][j] = 0.0f;
            }
        }
        if (valid < count) return;            // only masked positions follow
    }
}

// Runs that cross chunk borders: one CTA per (such run, column slice) adds its pieces, eight warps take consecutive ranges of
// them, and the eight sums are added in order.
template <typename Out, int kElems, bool kAccumulate>
__global__ void __launch_bounds__(256, 6) embedding_grad_join_kernel(const __grid_constant__ EmbGradArgs a) {
    using namespace emb_detail;
    __shared__ float sums[8][32 * kElems];
    const int lane = ptx::lane_id(), warp = threadIdx.x / 32;
    const int slices = math::ceil_div(a.hidden, 32 * kElems);
    cudaGridDependencySynchronize();          // launched before the sums are done
    const int64_t items = int64_t(*a.num_crossing) * slices;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int chunk = a.crossing[item / slices], slice = int(item % slices);
        const int id = a.ids[int64_t(chunk + 1) * a.chunk];
        // pieces: the chunks behind this one whose first position still belongs to the run, 32 looked at per step
        int pieces = 0;
        for (bool more = true; more; ) {
            const int c = chunk + 1 + pieces + lane;
            const unsigned same = __ballot_sync(0xffffffffu, c < a.num_chunks and a.ids[int64_t(c) * a.chunk] == id);
            pieces += __popc(same);
            more = same == 0xffffffffu;
        }
        const int per_warp = math::ceil_div(pieces, 8);
        const int first = min(warp * per_warp, pieces), last = min(first + per_warp, pieces);
        const int column = (slice * 32 + lane) * kElems;
        float acc[kElems];
        #pragma unroll
        for (int j = 0; j < kElems; ++j) acc[j] = 0.0f;
        if (column < a.hidden) {
            if (warp == 0) {
                unpack<float, kElems>(load_written_pack<float, kElems>(a.partial + (int64_t(chunk) * 2 + 1) * a.hidden + column), acc);
            }
            #pragma unroll 4
            for (int i = first; i < last; ++i) {
                float v[kElems];
                unpack<float, kElems>(load_written_pack<float, kElems>(a.partial + (int64_t(chunk + 1 + i) * 2) * a.hidden + column), v);
                #pragma unroll
                for (int j = 0; j < kElems; ++j) acc[j] += v[j];
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
            Out* out = reinterpret_cast<Out*>(a.out) + int64_t(id) * a.out_stride + column;
            if constexpr (kAccumulate) add_sum<kElems>(out, a.scale, acc, load_written_pack<float, kElems>(out));
            else write_sum<Out, kElems>(out, a.scale, acc);
        }
        __syncthreads();
    }
}

}  // namespace deep_ep::kernels
