// Low-rank adapters of many requests beside a shared projection, on sm_100a tensor cores:
//   y[i] = x[i] W^T + s_e (x[i] A_e^T) B_e^T      with e the adapter of row i,
// and the gradients dx = dy W + dt A_e, dA_e = dt^T x, dB_e = dy^T t with t = s_e x A_e^T and dt = s_e dy B_e.
//
// Three kernels, each with a TMA producer, one thread that issues `tcgen05.mma`, and accumulators in tensor memory:
//   lora_shrink   t (or dt): every row tile against the adapters that occur in it. Bound by reading x once.
//   lora_gemm     the shared product and the adapters' second product in ONE accumulator: the low-rank term is a few more
//                 K blocks of the same tile, so y is rounded once and neither product visits memory on the way. Bound by the
//                 tensor cores for many rows, by reading W for few.
//   lora_wgrad    dA, dB: contraction over the tokens of an adapter. Bound by reading x (dy) once.
//
// Rows keep the order in which they arrive; nothing is sorted or padded. In a tile with several adapters the rows of all
// but one are zeros in the A operand of an adapter's K block, so the K blocks of the adapters add up to the right rows.
// t enters the tensor cores as two bf16 numbers (its rounding and the rest), which keeps 16 of its bits: the low-rank
// product is as exact as its bf16 operands allow, at twice a cost that is a few percent of the shared product.
//
// Neither zeros nor a sum of two parts hide infinities or NaN (0 * inf = NaN, and so is hi * inf + lo * inf where lo is zero or of
// the other sign). lora_gemm therefore takes them out of both operands of an adapter's block and adds their products, in fp32, to the
// owner's rows (a NaN of t stays: its whole row of y is NaN); lora_wgrad overwrites the rows of other requests with zeros, and where the sum of hi's products is not finite that is
// the result. One request cannot poison another, and its own results are infinite or NaN where the formulas say so, whoever
// shares its tile.
#pragma once

#include "../device/sync.cuh"
#include "../device/tcgen05.cuh"
#include "lora_args.hpp"

namespace deep_ep::kernels {

namespace lora_detail {

constexpr int kNone = 0x7fffffff;

EP_DEVICE int adapter_of(const LoraRows& r, int row) {
    if (row >= r.num_rows) return -1;
    const int64_t id = r.idx64 ? reinterpret_cast<const int64_t*>(r.idx)[row] : reinterpret_cast<const int*>(r.idx)[row];
    return static_cast<uint64_t>(id) < static_cast<uint64_t>(r.num_adapters) ? static_cast<int>(id) : -1;
}

// The adapters of a tile's rows (128, or 256 for a pair of CTAs): enumerated in ascending order by minimum search, which needs
// no list, no sort and no other kernel.
template <int kRows>
struct TileAdapters {
    static constexpr int kPer = kRows / 32;
    int id[kPer];

    EP_DEVICE void load(const LoraRows& r, int m0, int lane) {
        #pragma unroll
        for (int i = 0; i < kPer; ++i) id[i] = adapter_of(r, m0 + lane + 32 * i);
    }
    EP_DEVICE int next(int last) const {
        unsigned best = kNone;
        #pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (id[i] > last) best = min(best, static_cast<unsigned>(id[i]));
        return static_cast<int>(__reduce_min_sync(0xffffffffu, best));
    }
};

EP_DEVICE bool has_non_finite(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    bool bad = false;
    #pragma unroll
    for (int i = 0; i < 4; ++i) bad = bad or (w[i] & 0x7f80u) == 0x7f80u or (w[i] & 0x7f800000u) == 0x7f800000u;
    return bad;
}

// t that the writers keep from the tensor cores: infinite, or infinite once it is rounded to bf16
EP_DEVICE bool taken_out(float t) { return isinf(__bfloat162float(__float2bfloat16_rn(t))); }
// v = hi + lo, both bf16. What is not finite has no lo, and with kTakeOut an infinity no hi either; true where there is one.
template <bool kTakeOut>
EP_DEVICE bool split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = ptx::float2_to_bf16x2(a, b);
    const float2 h = ptx::bf16x2_to_float2(hi);
    const float ra = a - h.x, rb = b - h.y;
    lo = ptx::float2_to_bf16x2(isfinite(ra) ? ra : 0.0f, isfinite(rb) ? rb : 0.0f);
    if constexpr (kTakeOut) {
        const bool ia = isinf(h.x), ib = isinf(h.y);
        hi &= (ia ? 0u : 0x0000ffffu) | (ib ? 0u : 0xffff0000u);
        return ia or ib;
    }
    return false;
}
// eight values -> one 16-byte unit each of hi and lo
template <bool kTakeOut>
EP_DEVICE bool split8(const float (&v)[8], uint4& hi, uint4& lo) {
    uint32_t h[4], l[4];
    bool found = false;
    #pragma unroll
    for (int i = 0; i < 4; ++i) found |= split2<kTakeOut>(v[2 * i], v[2 * i + 1], h[i], l[i]);
    hi = make_uint4(h[0], h[1], h[2], h[3]), lo = make_uint4(l[0], l[1], l[2], l[3]);
    return found;
}
EP_DEVICE void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

EP_DEVICE float4 ld_cluster_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
EP_DEVICE float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
EP_DEVICE int ld_cluster_int(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// Adds to v the products of a row's t and its adapter's V at columns n .. n + 7 (n a multiple of eight) that the writers have kept from
// the tensor cores: those of `taken_out` t, and of units of eight V elements with an infinity or NaN
__device__ __noinline__ void add_poisoned(const LoraGemmArgs& a, int row, int n, float (&v)[8]) {
    const int e = adapter_of(a.rows, row);
    if (e < 0) return;
    const __nv_bfloat16* base = reinterpret_cast<const __nv_bfloat16*>(a.v) + int64_t(e) * a.n * a.rows.rank;
    const float* t = a.t + int64_t(row) * a.rows.rank;
    float sum[8] = {};
    #pragma unroll 1
    for (int r = 0; r < a.rows.rank; r += 8) {
        float f[8];
        load8(t + r, f);
        unsigned out = 0;
        #pragma unroll
        for (int i = 0; i < 8; ++i) out |= unsigned(taken_out(f[i])) << i;
        // unit i: rank column r + i of the eight columns (mn_major), or eight rank columns of column n + i
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint4 u = *reinterpret_cast<const uint4*>(a.mn_major ? base + int64_t(r + i) * a.n + n : base + int64_t(n + i) * a.rows.rank + r);
            const unsigned which = has_non_finite(u) ? 0xffu : out;
            if (which == 0) continue;
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 g = ptx::bf16x2_to_float2(w[j / 2]);
                const float value = j % 2 ? g.y : g.x;
                if (a.mn_major and ((which >> i) & 1u)) sum[j] += f[i] * value;
                if (not a.mn_major and ((which >> j) & 1u)) sum[i] += f[j] * value;
            }
        }
        bool decided = true;                  // a NaN stays one (rows with several infinities get there at once)
        #pragma unroll
        for (int j = 0; j < 8; ++j) decided = decided and isnan(sum[j]);
        if (decided) break;
    }
    #pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += sum[j];
}

// This row's t, 32 columns from 32 * c (zeros behind the rank). Asked for a block ahead of its use: a read of a K block's own would be
// a round trip to L2 per block.
EP_DEVICE void read_t(const LoraGemmArgs& a, int row, bool there, int c, float (&t)[4][8]) {
    #pragma unroll
    for (int u = 0; u < 4; ++u) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) t[u][j] = 0.0f;
        if (there and 32 * c + 8 * u < a.rows.rank) load8(a.t + int64_t(row) * a.rows.rank + 32 * c + 8 * u, t[u]);
    }
}
// A row's line of an A slot: bf16 hi in the first half, lo in the second (zeros for rows of others), 16-byte unit u of row r at u ^ (r % 8).
// True where the row has a t that is taken out, which is written as zero.
EP_DEVICE bool write_t(uint8_t* slot, int row, bool there, const float (&t)[4][8]) {
    uint8_t* line = slot + row * 128;
    bool found = false;
    #pragma unroll
    for (int u = 0; u < 4; ++u) {
        uint4 hi = make_uint4(0, 0, 0, 0), lo = make_uint4(0, 0, 0, 0);
        if (there) found |= split8<true>(t[u], hi, lo);
        *reinterpret_cast<uint4*>(line + ((u ^ (row & 7)) << 4)) = hi;
        *reinterpret_cast<uint4*>(line + (((4 + u) ^ (row & 7)) << 4)) = lo;
    }
    return found;
}
// Takes infinities and NaN (whole units) out of the part of a V block of 128 columns that the products read: 32 columns of 128
// lines, or (mn_major) 32 lines of each of two blocks of 64 columns. 128 threads; true where this thread found one.
EP_DEVICE bool take_out_non_finite(uint8_t* block, bool mn_major, int thread) {
    constexpr int kUnits = 4;                 // per thread, read before any of them is looked at
    uint4* at[kUnits];
    uint4 unit[kUnits];
    #pragma unroll
    for (int q = 0; q < kUnits; ++q) {
        const int i = thread + q * 128;
        at[q] = reinterpret_cast<uint4*>(block + (mn_major ? (i / 256) * 8192 + (i % 256) * 16 : (i / 4) * 128 + (((i % 4) ^ ((i / 4) & 7)) << 4)));
        unit[q] = *at[q];
    }
    bool found = false;
    #pragma unroll
    for (int q = 0; q < kUnits; ++q)
        if (has_non_finite(unit[q])) *at[q] = make_uint4(0, 0, 0, 0), found = true;
    return found;
}

EP_DEVICE void store8(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(ptx::float2_to_bf16x2(v[0], v[1]), ptx::float2_to_bf16x2(v[2], v[3]),
                                              ptx::float2_to_bf16x2(v[4], v[5]), ptx::float2_to_bf16x2(v[6], v[7]));
}

// Epilogue of one warp: its 32 rows of an accumulator of `columns` columns, rounded to bf16 and stored by the TMA through a 4 KB
// buffer (what lies beyond the matrix is cut off by the store). `fix`: add what the tensor cores did not get.
EP_DEVICE void store_tile(const CUtensorMap* map_y, const LoraGemmArgs& a, uint32_t taddr, uint8_t* buffer, int row0, int n0, int columns, bool fix, int lane) {
    uint8_t* line = buffer + lane * 128;
    if (fix) cudaGridDependencySynchronize();
    for (int c = 0; c < columns; c += 64) {
        if (lane == 0) ptx::bulk_wait_read<0>();
        __syncwarp();
        if (not fix) {
            uint32_t lo[32], hi[32];
            tc::tmem_ld_32x32(taddr + c, lo);
            tc::tmem_ld_32x32(taddr + c + 32, hi);
            tc::wait_ld();
            #pragma unroll
            for (int u = 0; u < 4; ++u) {
                uint32_t w[4], w2[4];
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] = ptx::float2_to_bf16x2(__uint_as_float(lo[8 * u + 2 * j]), __uint_as_float(lo[8 * u + 2 * j + 1]));
                    w2[j] = ptx::float2_to_bf16x2(__uint_as_float(hi[8 * u + 2 * j]), __uint_as_float(hi[8 * u + 2 * j + 1]));
                }
                *reinterpret_cast<uint4*>(line + ((u ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                *reinterpret_cast<uint4*>(line + (((4 + u) ^ (lane & 7)) << 4)) = make_uint4(w2[0], w2[1], w2[2], w2[3]);
            }
        } else {
            #pragma unroll 1
            for (int u = 0; u < 8; ++u) {
                float v[8];
                #pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(tc::tmem_ld_32x1(taddr + c + 8 * u + j));
                tc::wait_ld();
                if (row0 + lane < a.rows.num_rows and n0 + c + 8 * u < a.n) add_poisoned(a, row0 + lane, n0 + c + 8 * u, v);
                __syncwarp();
                store8(reinterpret_cast<__nv_bfloat16*>(line + ((u ^ (lane & 7)) << 4)), v);
            }
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 and row0 < a.rows.num_rows and n0 + c < a.n) {
            tc::tma_store_2d(map_y, n0 + c, row0, buffer);
            ptx::bulk_commit();
        }
    }
}

// A row of the accumulator (`columns` fp32, a multiple of 32) to shared memory at `to`, possibly of another CTA of the cluster.
// Its 16-byte units are swizzled by the row, so that neither side has bank conflicts. Called by a whole warp.
EP_DEVICE void send_part(uint32_t to, uint32_t taddr, int columns, int row, bool valid) {
    for (int c = 0; c < columns; c += 32) {
        uint32_t r[32];
        tc::tmem_ld_32x32(taddr + c, r);
        tc::wait_ld();
        if (not valid) continue;
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};"
                         ::"r"(to + (((c / 4 + i) ^ (row & 7)) << 4)), "r"(r[4 * i]), "r"(r[4 * i + 1]), "r"(r[4 * i + 2]), "r"(r[4 * i + 3]) : "memory");
    }
}
// Adds columns c .. c + 7 of a row over the parts of all ranks, in rank order
EP_DEVICE void add_parts(float (&v)[8], const uint8_t* parts, int part_bytes, int ranks, int row_offset, int c, int row) {
    #pragma unroll 4
    for (int q = 0; q < ranks; ++q) {
        const uint8_t* line = parts + q * part_bytes + row_offset;
        const float4 x = *reinterpret_cast<const float4*>(line + (((c / 4) ^ (row & 7)) << 4));
        const float4 y = *reinterpret_cast<const float4*>(line + (((c / 4 + 1) ^ (row & 7)) << 4));
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
}

// One lane of a converged warp, always the same. The loops that feed the tensor cores are run by a whole warp and let this lane
// issue: their counters and descriptors then stay in uniform registers, which is what the instructions take. Run by a single
// lane of a diverged warp, a step of such a loop cost about twice as much.
EP_DEVICE bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
    return p != 0;
}
// Wait for a phase: false when somebody gave up (`error_flag`), or when this wait itself ran out (about 10 s), which sets the flag.
// The flag is looked at only when the barrier is not ready.
EP_DEVICE bool wait(uint64_t* bar, uint32_t parity, volatile int* error_flag) {
    if (ptx::mbarrier_try_wait(bar, parity)) return true;
    #pragma unroll 1
    for (int i = 0; i < 100; ++i) {
        if (*error_flag) return false;
        if (ptx::mbarrier_wait(bar, parity, 1 << 20, 100000000ull)) return true;
    }
    *error_flag = 1;
    return false;
}
EP_DEVICE bool wait_cluster(uint64_t* bar, uint32_t parity, volatile int* error_flag) {
    if (tc::mbarrier_try_wait_cluster(bar, parity)) return true;
    const unsigned long long start = ptx::globaltimer_ns();
    #pragma unroll 1
    while (not *error_flag) {
        #pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (tc::mbarrier_try_wait_cluster(bar, parity)) return true;
        if (ptx::globaltimer_ns() - start > 10000000000ull) *error_flag = 1;
    }
    return false;
}
EP_DEVICE bool wait_all_lanes(uint64_t* bar, uint32_t parity, volatile int* error_flag) {
    return __all_sync(0xffffffffu, wait(bar, parity, error_flag));
}
// this thread's copies into the last stages of a ring have landed
EP_DEVICE void drain(uint64_t* full_bar, int issued, int stages) {
    for (int i = max(0, issued - stages); i < issued; ++i) ptx::mbarrier_wait(&full_bar[i % stages], (i / stages) & 1);
}
// Position in a ring of stages
struct Ring {
    int slot = 0;
    uint32_t phase = 0;
    EP_DEVICE void advance(int stages) {
        if (++slot == stages) slot = 0, phase ^= 1;
    }
};

EP_DEVICE uint8_t* align_1024(uint8_t* p) { return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023)); }

EP_DEVICE void report(bool failed, int* status) {
    if (failed and status != nullptr) {
        *reinterpret_cast<volatile int*>(status) = 1;
        __threadfence_system();
    }
}

}  // namespace lora_detail

// ---------------------------------------------------------------------------------------- shrink
// A cluster owns (row tile, chunk of the tile's adapters); its CTAs share the contraction and add their sums through
// distributed shared memory in rank order. The accumulator holds the tile's rows against every adapter of the chunk
// (chunk * rank columns); each row picks the columns of its own. Rank <= 64 leaves the products far below the tensor
// cores' rate: what counts is that x is read once, by as many SMs as possible.
__global__ void __launch_bounds__(192, 1)
lora_shrink_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ LoraShrinkArgs a) {
    using namespace lora_detail;
    extern __shared__ uint8_t smem_raw[];
    constexpr int kMaxStages = 8;
    __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], done_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ int list[16], list_size;
    __shared__ volatile int error_flag;

    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) / 32, 0), lane = ptx::lane_id();
    const int cluster = a.cluster, rank = blockIdx.x % cluster;
    // (first chunks first: the later ones of most tiles are empty)
    const int tiles = math::ceil_div(a.rows.num_rows, kLoraTileRows), tile = int(blockIdx.x / cluster) % tiles, chunk = int(blockIdx.x / cluster) / tiles;
    const int m0 = tile * kLoraTileRows;
    // columns of the accumulator per adapter: the rank, padded (by zeros that the TMA fills in) to what the operand's layout has
    const int rp = math::align(a.rows.rank, a.mn_major ? 64 : 16);
    uint8_t* smem = align_1024(smem_raw);
    constexpr uint32_t kXBytes = kLoraTileRows * kLoraBlockK * 2;
    const uint32_t slot_bytes = rp * 128u;    // one adapter's block of a stage

    if (threadIdx.x == 0) {
        for (int s = 0; s < kMaxStages; ++s) ptx::mbarrier_init(&full_bar[s], 1), ptx::mbarrier_init(&empty_bar[s], 1);
        ptx::mbarrier_init(&done_bar, 1);
        ptx::fence_mbarrier_init();
        error_flag = 0;
        tc::prefetch_tensormap(&map_x), tc::prefetch_tensormap(&map_a);
    }
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    if (warp == 0) {
        // this chunk's adapters
        TileAdapters<kLoraTileRows> rows;
        rows.load(a.rows, m0, lane);
        int e = rows.next(-1);
        for (int i = 0; i < chunk * a.chunk and e != kNone; ++i) e = rows.next(e);
        int n = 0;
        for (; n < a.chunk and e != kNone; ++n, e = rows.next(e))
            if (lane == 0) list[n] = e;
        if (lane == 0) list_size = n;
    }
    if (a.presence != nullptr and chunk == 0 and rank == 0 and warp >= 2) {
        // for the weight gradients: which adapters occur in this row tile
        for (int e = warp - 2; e < a.rows.num_adapters; e += 4) {
            bool here = false;
            #pragma unroll
            for (int i = 0; i < 4; ++i) here = here or adapter_of(a.rows, m0 + lane + 32 * i) == e;
            here = __any_sync(0xffffffffu, here);
            if (lane == 0) a.presence[int64_t(tile) * a.rows.num_adapters + e] = here;
        }
    }
    __syncthreads();
    const int n = list_size;
    if (n == 0) return;                       // the same for all CTAs of the cluster
    // the ring is cut by the adapters that are there: fewer adapters, more stages in flight
    const int stage_bytes = int(kXBytes + n * slot_bytes), stages = min(kMaxStages, a.ring_bytes / stage_bytes);
    uint32_t columns = 32;
    while (columns < uint32_t(a.chunk * rp)) columns *= 2;
    if (warp == 1) tc::tmem_alloc(&tmem_slot, columns);
    tc::fence_before_thread_sync();
    __syncthreads();
    tc::fence_after_thread_sync();
    const uint32_t tmem = tmem_slot;

    const int blocks = math::ceil_div(a.k, kLoraBlockK), per = math::ceil_div(blocks, cluster);
    const int kb0 = min(rank * per, blocks), kb1 = min(kb0 + per, blocks);

    if (warp == 0) {
        Ring ring;
        int issued = 0;
        for (int kb = kb0; kb < kb1; ++kb, ++issued, ring.advance(stages)) {
            if (not wait_all_lanes(&empty_bar[ring.slot], ring.phase ^ 1, &error_flag)) break;
            if (elect_one()) {
                uint64_t* bar = &full_bar[ring.slot];
                uint8_t* stage = smem + size_t(ring.slot) * stage_bytes;
                ptx::mbarrier_arrive_expect_tx(bar, kXBytes + n * slot_bytes);
                tc::tma_load_2d(stage, &map_x, kb * kLoraBlockK, m0, bar);
                for (int j = 0; j < n; ++j) {
                    uint8_t* dst = stage + kXBytes + j * slot_bytes;
                    if (a.mn_major) {
                        for (int c = 0; c * 64 < rp; ++c) tc::tma_load_3d(dst + c * 8192, &map_a, c * 64, kb * kLoraBlockK, list[j], bar);
                    } else {
                        tc::tma_load_3d(dst, &map_a, kb * kLoraBlockK, 0, list[j], bar);
                    }
                }
            }
        }
        drain(full_bar, issued, stages);      // its own copies have landed before this warp leaves, also when somebody gave up
    } else if (warp == 1) {
        const uint32_t idesc = tc::make_idesc(tc::kFormatBF16, kLoraTileRows, rp, false, a.mn_major);
        const uint32_t b_lead = a.mn_major ? 8192 : 16, b_k = (a.mn_major ? 2048 : 32) >> 4;
        const uint64_t desc_x = tc::make_smem_desc(smem, 16, 1024), desc_a = tc::make_smem_desc(smem + kXBytes, b_lead, 1024);
        Ring ring;
        for (int kb = kb0; kb < kb1; ++kb, ring.advance(stages)) {
            wait(&full_bar[ring.slot], ring.phase, &error_flag);
            tc::fence_after_thread_sync();
            if (elect_one()) {
                const uint64_t step = uint64_t(ring.slot) * (stage_bytes >> 4);
                for (int j = 0; j < n; ++j) {
                    #pragma unroll
                    for (int k = 0; k < kLoraBlockK / 16; ++k)
                        tc::mma_f16(tmem + j * rp, desc_x + step + k * 2, desc_a + step + uint64_t(j) * (slot_bytes >> 4) + k * b_k, idesc, kb > kb0 or k > 0);
                }
                tc::commit(&empty_bar[ring.slot]);
            }
        }
        if (elect_one()) tc::commit(&done_bar);
    }
    // ---- every row picks its adapter's columns: straight to memory, or through shared memory and the cluster
    const int pitch = rp + 4;                 // floats per row of the staging area
    float* part = reinterpret_cast<float*>(smem);
    if (warp >= 2) {
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const int mine = adapter_of(a.rows, m0 + row);
        int slot = -1;
        for (int j = 0; j < n; ++j)
            if (list[j] == mine) slot = j;
        wait_all_lanes(&done_bar, 0, &error_flag);
        tc::fence_after_thread_sync();
        const float scale = slot >= 0 ? a.scaling[mine] : 0.0f;
        for (int j = 0; j < n; ++j) {
            if (not __any_sync(0xffffffffu, slot == j)) continue;
            for (int c = 0; c < a.rows.rank; c += 16) {
                uint32_t r[16];
                tc::tmem_ld_32x16(tmem + (uint32_t(quarter * 32) << 16) + j * rp + c, r);
                tc::wait_ld();
                if (slot != j) continue;
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 v = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]), __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
                    if (kb0 >= kb1) v = make_float4(0.f, 0.f, 0.f, 0.f);            // no K block fell to this CTA
                    if (cluster > 1) {
                        *reinterpret_cast<float4*>(part + row * pitch + c + 4 * i) = v;
                    } else if (c + 4 * i < a.rows.rank) {
                        *reinterpret_cast<float4*>(a.t + int64_t(m0 + row) * a.rows.rank + c + 4 * i) =
                            make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale);
                    }
                }
            }
        }
        tc::fence_before_thread_sync();
    }
    if (cluster > 1) {
        tc::cluster_sync();
        const int share = kLoraTileRows / cluster, units = a.rows.rank / 4;
        for (int item = threadIdx.x; item < share * units; item += 192) {
            const int row = rank * share + item / units, c = (item % units) * 4;
            const int mine = adapter_of(a.rows, m0 + row);
            bool here = false;
            for (int j = 0; j < n; ++j) here = here or list[j] == mine;
            if (not here) continue;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int q = 0; q < cluster; ++q) {
                const float4 v = ld_cluster_v4(tc::map_to_cta(part + row * pitch + c, q));
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
            const float scale = a.scaling[mine];
            *reinterpret_cast<float4*>(a.t + int64_t(m0 + row) * a.rows.rank + c) = make_float4(sum.x * scale, sum.y * scale, sum.z * scale, sum.w * scale);
        }
        tc::cluster_sync();                   // nobody leaves while others read its shared memory
    }
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_thread_sync();
        tc::tmem_dealloc(tmem, columns);
    }
    if (threadIdx.x == 0) report(error_flag != 0, a.rows.status);
}

// The same for a few rows (decode): one CTA per (row, four rank columns), plain fp32 products. A tile of the kernel above would
// be mostly empty, and its setup (tensor maps, tensor memory, a cluster) costs more than these products; the adapters are
// read once per row, from L2. Its time is that of round trips to memory, those for its instructions among them: between two
// calls a decode step streams more weights than L2 holds, so the code is cold. Hence a short loop instead of an unrolled one
// (which took 8.6 us for one row of 7168, of which 5 went to fetching instructions). Small CTAs: three of them and one of the
// kernel that reads W fit on an SM together, so that W is under way while these wait.
__global__ void __launch_bounds__(256, 6)
lora_shrink_rows_kernel(const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ a_all, const __grid_constant__ LoraShrinkArgs a) {
    using namespace lora_detail;
    constexpr int kColumns = 4, kThreads = 256;
    __shared__ float sums[kThreads / 32][kColumns];
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    const int groups = a.rows.rank / kColumns, row = blockIdx.x / groups, r0 = blockIdx.x % groups * kColumns;
    const int warp = threadIdx.x / 32, lane = ptx::lane_id();
    const int e = adapter_of(a.rows, row);
    if (a.presence != nullptr and r0 == 0 and row % kLoraTileRows == 0) {
        for (int p = warp; p < a.rows.num_adapters; p += kThreads / 32) {
            bool here = false;
            #pragma unroll 1
            for (int i = 0; i < 4; ++i) here = here or adapter_of(a.rows, row + lane + 32 * i) == p;
            here = __any_sync(0xffffffffu, here);
            if (lane == 0) a.presence[int64_t(row / kLoraTileRows) * a.rows.num_adapters + p] = here;
        }
    }
    if (e < 0) return;
    const float scale = a.scaling[e];
    const __nv_bfloat16* xr = x + int64_t(row) * a.k;
    const __nv_bfloat16* ae = a_all + int64_t(e) * a.rows.rank * a.k;
    float acc[kColumns] = {};
    if (a.mn_major) {
        // A_e [k, rank]: a thread takes single k with the columns of this CTA
        #pragma unroll 2
        for (int k = threadIdx.x; k < a.k; k += kThreads) {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(ae + int64_t(k) * a.rows.rank + r0));
            const float v = __bfloat162float(xr[k]);
            const float2 f = ptx::bf16x2_to_float2(u.x), g = ptx::bf16x2_to_float2(u.y);
            acc[0] = fmaf(v, f.x, acc[0]), acc[1] = fmaf(v, f.y, acc[1]), acc[2] = fmaf(v, g.x, acc[2]), acc[3] = fmaf(v, g.y, acc[3]);
        }
    } else {
        // A_e [rank, k]: a thread takes eight k of each of the rows
        ae += int64_t(r0) * a.k;
        #pragma unroll 1
        for (int k = threadIdx.x * 8; k < a.k; k += kThreads * 8) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(xr + k));
            uint4 v[kColumns];
            #pragma unroll
            for (int r = 0; r < kColumns; ++r) v[r] = __ldg(reinterpret_cast<const uint4*>(ae + int64_t(r) * a.k + k));
            const uint32_t xw[4] = {u.x, u.y, u.z, u.w};
            #pragma unroll
            for (int r = 0; r < kColumns; ++r) {
                const uint32_t w[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
                #pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float2 f = ptx::bf16x2_to_float2(w[q]), g = ptx::bf16x2_to_float2(xw[q]);
                    acc[r] = fmaf(g.x, f.x, acc[r]), acc[r] = fmaf(g.y, f.y, acc[r]);
                }
            }
        }
    }
    // four sums over 32 lanes: two steps halve the number of sums a lane carries (lane bits 4 and 3 say which), three add the rest
    const bool upper = lane & 16, odd = lane & 8;
    const float p0 = (upper ? acc[2] : acc[0]) + __shfl_xor_sync(0xffffffffu, upper ? acc[0] : acc[2], 16);
    const float p1 = (upper ? acc[3] : acc[1]) + __shfl_xor_sync(0xffffffffu, upper ? acc[1] : acc[3], 16);
    float sum = (odd ? p1 : p0) + __shfl_xor_sync(0xffffffffu, odd ? p0 : p1, 8);
    #pragma unroll
    for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane % 8 == 0) sums[warp][lane / 8] = sum;
    __syncthreads();
    if (threadIdx.x < kColumns) {
        float total = 0.0f;
        #pragma unroll 4
        for (int w = 0; w < kThreads / 32; ++w) total += sums[w][threadIdx.x];
        a.t[int64_t(row) * a.rows.rank + r0 + threadIdx.x] = total * scale;
    }
}

// ---------------------------------------------------------------------------------------- shared product + adapters
// Tiles of 128 rows x BN columns.
//   warp 0      TMA producer: K blocks of x and W, then the V blocks of the tile's adapters
//   warp 1      MMA issuer
//   warps 2-5   epilogue
//   warps 6-13  writers: the A operand of the adapters' K blocks (t as bf16 hi | lo, zeros in the rows of others), two groups that
//               take the blocks in turn: a block takes a group about a microsecond, the tensor cores a third of that (2048 rows
//               of 8 adapters of rank 64, K and N 4096: 101 us, 123 with one group)
// Many tiles: persistent CTAs, two accumulators in tensor memory, so that the stores of one tile overlap the products of the
// next. Few tiles (decode): a cluster shares the tile's contraction, so that all SMs pull on W; its CTAs send their parts
// of a row to the CTA that owns the row, which adds them in rank order.
constexpr int kLoraGemmColumns = 128, kLoraGemmStages = 5, kLoraGemmThreads = 448;
constexpr int kLoraGemmSmemBytes = kLoraGemmStages * (kLoraTileRows + kLoraGemmColumns) * kLoraBlockK * 2 + kLoraTileRows * kLoraGemmColumns * 4 + 1024;

__global__ void __launch_bounds__(kLoraGemmThreads, 1)
lora_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap map_y, const __grid_constant__ LoraGemmArgs a) {
    using namespace lora_detail;
    extern __shared__ uint8_t smem_raw[];
    constexpr int BN = kLoraGemmColumns, kStages = kLoraGemmStages, kGroupM = 16;
    constexpr uint32_t kABytes = kLoraTileRows * kLoraBlockK * 2, kBBytes = BN * kLoraBlockK * 2;
    constexpr int kPoisonSlots = 8;           // more tiles than the writers can be ahead of the epilogue
    __shared__ uint64_t full_bar[kStages], empty_bar[kStages], grant_bar[2][kStages], ext_bar[kStages], tmem_full_bar[2], tmem_empty_bar[2];
    __shared__ uint64_t list_full_bar[2], list_empty_bar[2];
    __shared__ int list[2][kLoraTileRows], list_size[2];       // the adapters of a tile
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int error_flag, poison[kPoisonSlots];

    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) / 32, 0), lane = ptx::lane_id();
    const int cluster = a.cluster, rank = cluster > 1 ? int(blockIdx.x) % cluster : 0;
    const int num_tiles = a.m_tiles * a.n_tiles;
    const int first_tile = int(blockIdx.x) / cluster, tile_step = int(gridDim.x) / cluster;
    const bool split = cluster > 1;                            // parts are exchanged; one tile per cluster
    uint8_t* smem_a = align_1024(smem_raw);
    uint8_t* smem_b = smem_a + kStages * kABytes;
    uint8_t* smem_out = smem_b + kStages * kBBytes;            // a chunk of 32 rows x 64 columns per epilogue warp, or the parts

    const int blocks = math::ceil_div(a.k, kLoraBlockK), per = math::ceil_div(blocks, cluster);
    const int kb0 = min(rank * per, blocks), kb1 = min(kb0 + per, blocks);        // never empty, see the launcher
    const int rank_chunks = math::ceil_div(a.rows.rank, 32);                      // 32 rank columns (hi and lo) per K block

    // tile -> origin; groups of 16 row tiles run through all columns, so that their rows of x and all of W stay in L2
    const auto origin = [&](int tile, int& m0, int& n0) {
        const int group = tile / (kGroupM * a.n_tiles), first_m = group * kGroupM, gm = min(kGroupM, a.m_tiles - first_m);
        const int local = tile - group * kGroupM * a.n_tiles;
        m0 = (first_m + local % gm) * kLoraTileRows, n0 = local / gm * BN;
    };
    const auto load_block = [&](unsigned s, int m0, int n0, int kb) {
        ptx::mbarrier_arrive_expect_tx(&full_bar[s], kABytes + kBBytes);
        const int k0 = kb * kLoraBlockK;
        tc::tma_load_2d(smem_a + s * kABytes, &map_x, k0, m0, &full_bar[s]);
        uint8_t* sb = smem_b + s * kBBytes;
        if (a.mn_major) {
            #pragma unroll
            for (int i = 0; i < BN / 64; ++i) tc::tma_load_2d(sb + i * 8192, &map_w, n0 + 64 * i, k0, &full_bar[s]);
        } else {
            #pragma unroll
            for (int i = 0; i < BN / 128; ++i) tc::tma_load_2d(sb + i * 16384, &map_w, k0, n0 + 128 * i, &full_bar[s]);
        }
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s)
            ptx::mbarrier_init(&full_bar[s], 1), ptx::mbarrier_init(&empty_bar[s], 1), ptx::mbarrier_init(&grant_bar[0][s], 1), ptx::mbarrier_init(&grant_bar[1][s], 1), ptx::mbarrier_init(&ext_bar[s], 4);
        for (int i = 0; i < 2; ++i) {
            ptx::mbarrier_init(&tmem_full_bar[i], 1), ptx::mbarrier_init(&tmem_empty_bar[i], 4);
            ptx::mbarrier_init(&list_full_bar[i], 1), ptx::mbarrier_init(&list_empty_bar[i], 10);
        }
        ptx::fence_mbarrier_init();
        error_flag = 0;
        for (int i = 0; i < kPoisonSlots; ++i) poison[i] = 0;
    }
    if (threadIdx.x == 64) tc::prefetch_tensormap(&map_x), tc::prefetch_tensormap(&map_w), tc::prefetch_tensormap(&map_v), tc::prefetch_tensormap(&map_y);
    if (warp == 1) tc::tmem_alloc(&tmem_slot, split ? BN : 2 * BN);
    tc::fence_before_thread_sync();
    __syncthreads();
    tc::fence_after_thread_sync();
    const uint32_t tmem = tmem_slot;
    if (split) tc::cluster_arrive();          // (waited for before the first access to another CTA's shared memory)

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        Ring ring;
        int issued = 0, local = 0;
        unsigned ext = 0;                     // adapters' blocks so far
        bool ok = true;
        for (int tile = first_tile; tile < num_tiles and ok; tile += tile_step, ++local) {
            int m0, n0;
            origin(tile, m0, n0);
            for (int kb = kb0; kb < kb1 and ok; ++kb) {
                ok = wait_all_lanes(&empty_bar[ring.slot], ring.phase ^ 1, &error_flag);
                if (not ok) break;
                if (elect_one()) load_block(ring.slot, m0, n0, kb);
                ++issued, ring.advance(kStages);
            }
            const int slot = local & 1;
            ok = ok and wait_all_lanes(&list_full_bar[slot], (local >> 1) & 1, &error_flag);
            if (not ok) break;
            const int size = list_size[slot];
            for (int i = rank; i < size and ok; i += cluster) {
                const int e = list[slot][i];
                for (int c = 0; c < rank_chunks; ++c) {
                    ok = wait_all_lanes(&empty_bar[ring.slot], ring.phase ^ 1, &error_flag);
                    if (not ok) break;
                    if (elect_one()) {
                        uint64_t* bar = &full_bar[ring.slot];
                        ptx::mbarrier_arrive(&grant_bar[ext & 1][ring.slot]);    // the writers may fill the A slot
                        ptx::mbarrier_arrive_expect_tx(bar, kBBytes);
                        uint8_t* sb = smem_b + ring.slot * kBBytes;
                        if (a.mn_major) {
                            #pragma unroll
                            for (int j = 0; j < BN / 64; ++j) tc::tma_load_3d(sb + j * 8192, &map_v, n0 + 64 * j, 32 * c, e, bar);
                        } else {
                            #pragma unroll
                            for (int j = 0; j < BN / 128; ++j) tc::tma_load_3d(sb + j * 16384, &map_v, 32 * c, n0 + 128 * j, e, bar);
                        }
                    }
                    ++issued, ++ext, ring.advance(kStages);
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbarrier_arrive(&list_empty_bar[slot]);
        }
        drain(full_bar, issued, kStages);     // its own copies have landed before this warp leaves, also when somebody gave up
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        const uint32_t idesc = tc::make_idesc(tc::kFormatBF16, kLoraTileRows, BN, false, a.mn_major);
        const uint32_t b_lead = a.mn_major ? 8192 : 16, b_k = (a.mn_major ? 2048 : 32) >> 4;
        const uint64_t desc_a0 = tc::make_smem_desc(smem_a, 16, 1024), desc_b0 = tc::make_smem_desc(smem_b, b_lead, 1024);
        Ring ring;
        unsigned ext_phase = 0;
        int local = 0;
        for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++local) {
            const int acc = local & 1, slot = local & 1;
            const uint32_t d = tmem + acc * BN;
            wait(&tmem_empty_bar[acc], ((local >> 1) & 1) ^ 1, &error_flag);
            tc::fence_after_thread_sync();
            for (int kb = kb0; kb < kb1; ++kb, ring.advance(kStages)) {
                wait(&full_bar[ring.slot], ring.phase, &error_flag);
                tc::fence_after_thread_sync();
                if (elect_one()) {
                    const uint64_t da = desc_a0 + uint64_t(ring.slot * (kABytes >> 4)), db = desc_b0 + uint64_t(ring.slot * (kBBytes >> 4));
                    #pragma unroll
                    for (int k = 0; k < kLoraBlockK / 16; ++k) tc::mma_f16(d, da + k * 2, db + k * b_k, idesc, kb > kb0 or k > 0);
                    tc::commit(&empty_bar[ring.slot]);
                }
            }
            const int size = wait_all_lanes(&list_full_bar[slot], (local >> 1) & 1, &error_flag) ? list_size[slot] : 0;
            __syncwarp();
            if (lane == 0) ptx::mbarrier_arrive(&list_empty_bar[slot]);
            for (int i = rank; i < size; i += cluster) {
                for (int c = 0; c < rank_chunks; ++c, ring.advance(kStages)) {
                    wait(&full_bar[ring.slot], ring.phase, &error_flag);
                    wait(&ext_bar[ring.slot], (ext_phase >> ring.slot) & 1, &error_flag);
                    ext_phase ^= 1u << ring.slot;
                    tc::fence_after_thread_sync();
                    if (elect_one()) {
                        const uint64_t da = desc_a0 + uint64_t(ring.slot * (kABytes >> 4)), db = desc_b0 + uint64_t(ring.slot * (kBBytes >> 4));
                        for (int k = 0; k < 2 and 32 * c + 16 * k < a.rows.rank; ++k) {
                            tc::mma_f16(d, da + k * 2, db + k * b_k, idesc, true);             // hi
                            tc::mma_f16(d, da + 4 + k * 2, db + k * b_k, idesc, true);         // lo
                        }
                        tc::commit(&empty_bar[ring.slot]);
                    }
                }
            }
            if (elect_one()) tc::commit(&tmem_full_bar[acc]);
        }
    } else if (warp >= 6) {
        // ------------------------------------------------------------------ writers of the adapters' A operand
        cudaGridDependencySynchronize();      // t comes from the kernel before, which this one does not wait for until here
        const int row = (threadIdx.x - 192) & 127;
        const unsigned group = (warp - 6) / 4;
        // These warps do not follow the ring through the K blocks of x, so they cannot tell from a slot's own barriers (which
        // show a phase's parity only) whether it is free for THIS block: the producer, which can, grants it (on barriers of the
        // group's own, of which it thus misses no phase).
        unsigned it = 0, ext = 0, granted = 0;
        int local = 0;
        bool ok = true;
        for (int tile = first_tile; tile < num_tiles and ok; tile += tile_step, ++local) {
            int m0, n0;
            origin(tile, m0, n0);
            const int mine = adapter_of(a.rows, m0 + row), slot = local & 1;
            if (warp == 6) {
                // the tile's adapters for the producer and the MMA issuer
                TileAdapters<kLoraTileRows> rows;
                rows.load(a.rows, m0, lane);
                ok = wait_all_lanes(&list_empty_bar[slot], ((local >> 1) & 1) ^ 1, &error_flag);
                int size = 0;
                for (int e = rows.next(-1); e != kNone; e = rows.next(e), ++size)
                    if (lane == 0) list[slot][size] = e;
                if (lane == 0) list_size[slot] = size;
                if (not ok) break;
                if (lane == 0) ptx::mbarrier_arrive(&list_full_bar[slot]);
            }
            it += kb1 - kb0;
            // this group's first chunk of the row's t (exact when the chunks are even in number) is read before the ring has room for it
            int held = rank_chunks % 2 == 0 and (ext & 1) != group ? 1 : 0;
            float t[4][8];
            read_t(a, m0 + row, mine >= 0, held, t);
            ok = wait_all_lanes(&list_full_bar[slot], (local >> 1) & 1, &error_flag);
            if (not ok) break;
            const int size = list_size[slot];
            for (int i = rank; i < size and ok; i += cluster) {
                const int e = list[slot][i];
                for (int c = 0; c < rank_chunks; ++c, ++it, ++ext) {
                    if ((ext & 1) != group) continue;
                    const unsigned s = it % kStages, phase = (it / kStages) & 1;
                    if (mine == e and held != c) read_t(a, m0 + row, true, c, t);
                    ok = wait_all_lanes(&grant_bar[group][s], (granted >> s) & 1, &error_flag);
                    granted ^= 1u << s;
                    if (not ok) break;
                    bool found = write_t(smem_a + s * kABytes, row, mine == e, t);
                    if (mine == e and c + 2 < rank_chunks) held = c + 2, read_t(a, m0 + row, true, held, t);
                    ok = wait_all_lanes(&full_bar[s], phase, &error_flag);
                    if (not ok) break;
                    found |= take_out_non_finite(smem_b + s * kBBytes, a.mn_major, row);
                    if (found) poison[local % kPoisonSlots] = local + 1;
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) ptx::mbarrier_arrive(&ext_bar[s]);
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbarrier_arrive(&list_empty_bar[slot]);
        }
    }

    if (warp >= 2 and warp < 6) {
        // ------------------------------------------------------------------ epilogue
        const int quarter = warp & 3, row = quarter * 32 + lane;
        uint8_t* buffer = smem_out + quarter * 4096;
        int local = 0;
        for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++local) {
            int m0, n0;
            origin(tile, m0, n0);
            const int acc = local & 1;
            if (not wait_all_lanes(&tmem_full_bar[acc], (local >> 1) & 1, &error_flag)) {
                if (split) tc::cluster_wait();
                break;
            }
            tc::fence_after_thread_sync();
            const uint32_t taddr = tmem + acc * BN + (uint32_t(quarter * 32) << 16);
            if (split) {
                tc::cluster_wait();
                // fp32 parts to the CTA that owns the row: [rank][row][column], 16-byte units swizzled by the row
                if (m0 + quarter * 32 < a.rows.num_rows) {
                    const int share = kLoraTileRows / cluster;
                    send_part(tc::map_to_cta(smem_out + (rank * share + row % share) * (BN * 4), row / share), taddr, BN, row, m0 + row < a.rows.num_rows);
                }
                tc::fence_before_thread_sync();
                break;                        // one tile per cluster
            }
            store_tile(&map_y, a, taddr, buffer, m0 + quarter * 32, n0, BN, poison[local % kPoisonSlots] == local + 1, lane);
            tc::fence_before_thread_sync();
            __syncwarp();
            if (lane == 0) ptx::mbarrier_arrive(&tmem_empty_bar[acc]);
        }
        if (lane == 0) ptx::bulk_wait<0>();
        __syncwarp();
    }

    if (split) {
        // ------------------------------------------------------------------ sum of the parts
        int m0, n0;
        origin(first_tile, m0, n0);
        const int share = kLoraTileRows / cluster;
        __syncwarp();
        if (warp < 2 or warp >= 6) tc::cluster_wait();         // (the epilogue warps have done so)
        tc::cluster_sync();
        bool fix = false;
        for (int q = 0; q < cluster; ++q) fix = fix or ld_cluster_int(tc::map_to_cta(const_cast<const int*>(&poison[0]), q)) != 0;
        if (fix) cudaGridDependencySynchronize();
        for (int item = threadIdx.x; item < share * (BN / 8); item += kLoraGemmThreads) {
            const int row = rank * share + item / (BN / 8), c = item % (BN / 8) * 8;
            if (m0 + row >= a.rows.num_rows or n0 + c >= a.n) continue;
            float v[8] = {};
            add_parts(v, smem_out, share * BN * 4, cluster, (row % share) * BN * 4, c, row);
            if (fix) add_poisoned(a, m0 + row, n0 + c, v);
            store8(reinterpret_cast<__nv_bfloat16*>(a.y) + int64_t(m0 + row) * a.n + n0 + c, v);
        }
        tc::cluster_sync();                   // nobody leaves while others look at its flag
    }

    tc::fence_before_thread_sync();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_thread_sync();
        tc::tmem_dealloc(tmem, split ? BN : 2 * BN);
    }
    if (threadIdx.x == 0) report(error_flag != 0, a.rows.status);
}

// The same by pairs of CTAs (`cta_group::2`) for many tiles: 256 x 256 per pair, each CTA with its 128 rows of A, half of the 256
// columns of B, and the accumulator of its rows. A CTA alone reads 12 KB of shared memory for the products of a K step of 16 and
// takes in as much from the TMA: 192 bytes per clock, where shared memory has 128. A pair needs a third less per SM. Measured
// with K 4096, N 4096, rank 16: 115 / 209 us for 4096 / 8192 rows, 128 x 128 tiles by single CTAs 139 / 300 us.
// The MMAs are issued by the even CTA; barriers that concern it count both CTAs. A V block lands on a barrier of its own CTA,
// where the writers look at it; the even CTA learns from the writers of both that the block is complete.
constexpr int kLoraPairStages = 6;
constexpr int kLoraPairSmemBytes = kLoraPairStages * 2 * 128 * kLoraBlockK * 2 + 4 * 4096 + 1024;

__global__ void __launch_bounds__(kLoraGemmThreads, 1)
lora_gemm_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ CUtensorMap map_y, const __grid_constant__ LoraGemmArgs a) {
    using namespace lora_detail;
    extern __shared__ uint8_t smem_raw[];
    constexpr int kStages = kLoraPairStages, kGroupM = 8, kPoisonSlots = 8;
    constexpr uint32_t kHalf = 128 * kLoraBlockK * 2;          // 128 rows of A, or 128 columns of B: 16 KB
    __shared__ uint64_t full_bar[kStages], empty_bar[kStages], v_bar[2][kStages], ext_bar[kStages], tmem_full_bar[2], tmem_empty_bar[2];
    __shared__ uint64_t list_full_bar[2], list_empty_bar[2];
    __shared__ int list[2][2 * kLoraTileRows], list_size[2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int error_flag, poison[kPoisonSlots];

    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) / 32, 0), lane = ptx::lane_id();
    const int half = int(tc::cluster_ctarank());               // 0: even CTA, issues the MMAs
    const bool leader = half == 0;
    const int num_tiles = a.m_tiles * a.n_tiles, first_tile = int(blockIdx.x) / 2, tile_step = int(gridDim.x) / 2;
    const int blocks = math::ceil_div(a.k, kLoraBlockK), rank_chunks = math::ceil_div(a.rows.rank, 32);
    uint8_t* smem_a = align_1024(smem_raw);
    uint8_t* smem_b = smem_a + kStages * kHalf;
    uint8_t* smem_out = smem_b + kStages * kHalf;

    // tile -> origin, see above
    const auto origin = [&](int tile, int& m0, int& n0) {
        const int group = tile / (kGroupM * a.n_tiles), first_m = group * kGroupM, gm = min(kGroupM, a.m_tiles - first_m);
        const int local = tile - group * kGroupM * a.n_tiles;
        m0 = (first_m + local % gm) * 2 * kLoraTileRows, n0 = local / gm * 256;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s)
            ptx::mbarrier_init(&full_bar[s], 1), ptx::mbarrier_init(&empty_bar[s], 1), ptx::mbarrier_init(&v_bar[0][s], 1), ptx::mbarrier_init(&v_bar[1][s], 1), ptx::mbarrier_init(&ext_bar[s], 8);
        for (int i = 0; i < 2; ++i) {
            ptx::mbarrier_init(&tmem_full_bar[i], 1), ptx::mbarrier_init(&tmem_empty_bar[i], 8);
            ptx::mbarrier_init(&list_full_bar[i], 1), ptx::mbarrier_init(&list_empty_bar[i], leader ? 10 : 9);
        }
        ptx::fence_mbarrier_init();
        error_flag = 0;
        for (int i = 0; i < kPoisonSlots; ++i) poison[i] = 0;
    }
    if (threadIdx.x == 64) tc::prefetch_tensormap(&map_x), tc::prefetch_tensormap(&map_w), tc::prefetch_tensormap(&map_v), tc::prefetch_tensormap(&map_y);
    __syncthreads();
    tc::cluster_sync();                       // both CTAs' barriers exist before anyone signals across the pair
    if (warp == 1) tc::tmem_alloc_pair(&tmem_slot, 512);
    tc::fence_before_thread_sync();
    __syncthreads();
    tc::fence_after_thread_sync();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer (both CTAs)
        Ring ring;
        int issued = 0, local = 0;
        unsigned ext = 0;                     // adapters' blocks so far
        bool ok = true;
        for (int tile = first_tile; tile < num_tiles and ok; tile += tile_step, ++local) {
            int m0, n0;
            origin(tile, m0, n0);
            const int m_half = m0 + 128 * half, n_half = n0 + 128 * half;
            for (int kb = 0; kb < blocks; ++kb) {
                ok = wait_all_lanes(&empty_bar[ring.slot], ring.phase ^ 1, &error_flag);
                if (not ok) break;
                if (elect_one()) {
                    // the bytes of both CTAs are counted on the even CTA's barrier
                    const uint32_t bar = tc::map_to_cta(&full_bar[ring.slot], 0);
                    if (leader) ptx::mbarrier_arrive_expect_tx(&full_bar[ring.slot], 4 * kHalf);
                    const int k0 = kb * kLoraBlockK;
                    uint8_t* sb = smem_b + ring.slot * kHalf;
                    tc::tma_load_2d_pair(smem_a + ring.slot * kHalf, &map_x, k0, m_half, bar);
                    if (a.mn_major) {
                        tc::tma_load_2d_pair(sb, &map_w, n_half, k0, bar);
                        tc::tma_load_2d_pair(sb + 8192, &map_w, n_half + 64, k0, bar);
                    } else {
                        tc::tma_load_2d_pair(sb, &map_w, k0, n_half, bar);
                    }
                }
                ++issued, ring.advance(kStages);
            }
            const int slot = local & 1;
            ok = ok and wait_all_lanes(&list_full_bar[slot], (local >> 1) & 1, &error_flag);
            if (not ok) break;
            const int size = list_size[slot];
            for (int i = 0; i < size and ok; ++i) {
                const int e = list[slot][i];
                for (int c = 0; c < rank_chunks; ++c) {
                    ok = wait_all_lanes(&empty_bar[ring.slot], ring.phase ^ 1, &error_flag);
                    if (not ok) break;
                    if (elect_one()) {
                        uint64_t* bar = &v_bar[ext & 1][ring.slot];
                        ptx::mbarrier_arrive_expect_tx(bar, kHalf);
                        uint8_t* sb = smem_b + ring.slot * kHalf;
                        if (a.mn_major) {
                            tc::tma_load_3d(sb, &map_v, n_half, 32 * c, e, bar);
                            tc::tma_load_3d(sb + 8192, &map_v, n_half + 64, 32 * c, e, bar);
                        } else {
                            tc::tma_load_3d(sb, &map_v, 32 * c, n_half, e, bar);
                        }
                    }
                    ++issued, ++ext, ring.advance(kStages);
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbarrier_arrive(&list_empty_bar[slot]);
        }
        // what this CTA asked for has landed, and been read by the MMAs, before it leaves (a bounded wait also when somebody gave up)
        for (int i = max(0, issued - kStages); i < issued; ++i) ptx::mbarrier_wait(&empty_bar[i % kStages], (i / kStages) & 1);
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer (even CTA only)
        const uint32_t idesc = tc::make_idesc(tc::kFormatBF16, 256, 256, false, a.mn_major);
        const uint32_t b_lead = a.mn_major ? 8192 : 16, b_k = (a.mn_major ? 2048 : 32) >> 4;
        const uint64_t desc_a0 = tc::make_smem_desc(smem_a, 16, 1024), desc_b0 = tc::make_smem_desc(smem_b, b_lead, 1024);
        Ring ring;
        unsigned full_phase = 0, ext_phase = 0;       // per slot: a slot's blocks of x and of V complete on different barriers
        int local = 0;
        for (int tile = leader ? first_tile : num_tiles; tile < num_tiles; tile += tile_step, ++local) {
            const int acc = local & 1, slot = local & 1;
            const uint32_t d = tmem + acc * 256;
            wait_cluster(&tmem_empty_bar[acc], ((local >> 1) & 1) ^ 1, &error_flag);
            tc::fence_after_thread_sync();
            for (int kb = 0; kb < blocks; ++kb, ring.advance(kStages)) {
                wait(&full_bar[ring.slot], (full_phase >> ring.slot) & 1, &error_flag);
                full_phase ^= 1u << ring.slot;
                tc::fence_after_thread_sync();
                if (elect_one()) {
                    const uint64_t da = desc_a0 + uint64_t(ring.slot * (kHalf >> 4)), db = desc_b0 + uint64_t(ring.slot * (kHalf >> 4));
                    #pragma unroll
                    for (int k = 0; k < kLoraBlockK / 16; ++k) tc::mma_f16_pair(d, da + k * 2, db + k * b_k, idesc, kb > 0 or k > 0);
                    tc::commit_pair(&empty_bar[ring.slot]);    // the stage is free in both CTAs once these MMAs have read it
                }
            }
            const int size = wait_all_lanes(&list_full_bar[slot], (local >> 1) & 1, &error_flag) ? list_size[slot] : 0;
            __syncwarp();
            if (lane == 0) ptx::mbarrier_arrive(&list_empty_bar[slot]);
            for (int i = 0; i < size * rank_chunks; ++i, ring.advance(kStages)) {
                const int c = i % rank_chunks;
                wait_cluster(&ext_bar[ring.slot], (ext_phase >> ring.slot) & 1, &error_flag);
                ext_phase ^= 1u << ring.slot;
                tc::fence_after_thread_sync();
                if (elect_one()) {
                    const uint64_t da = desc_a0 + uint64_t(ring.slot * (kHalf >> 4)), db = desc_b0 + uint64_t(ring.slot * (kHalf >> 4));
                    for (int k = 0; k < 2 and 32 * c + 16 * k < a.rows.rank; ++k) {
                        tc::mma_f16_pair(d, da + k * 2, db + k * b_k, idesc, true);             // hi
                        tc::mma_f16_pair(d, da + 4 + k * 2, db + k * b_k, idesc, true);         // lo
                    }
                    tc::commit_pair(&empty_bar[ring.slot]);
                }
            }
            if (elect_one()) tc::commit_pair(&tmem_full_bar[acc]);
        }
    } else if (warp >= 6) {
        // ------------------------------------------------------------------ writers of the adapters' A operand (both CTAs, own rows)
        cudaGridDependencySynchronize();      // t comes from the kernel before, which this one does not wait for until here
        const int row = (threadIdx.x - 192) & 127;
        const unsigned group = (warp - 6) / 4;
        unsigned landed = 0, ext = 0;         // per slot: parity of this group's next V block; blocks so far
        int position = 0, local = 0;          // position in the ring
        bool ok = true;
        for (int tile = first_tile; tile < num_tiles and ok; tile += tile_step, ++local) {
            int m0, n0;
            origin(tile, m0, n0);
            const int my_row = m0 + 128 * half + row, mine = adapter_of(a.rows, my_row), slot = local & 1;
            if (warp == 6) {
                // the adapters of the pair's 256 rows, for the producer and the MMA issuer
                TileAdapters<2 * kLoraTileRows> rows;
                rows.load(a.rows, m0, lane);
                ok = wait_all_lanes(&list_empty_bar[slot], ((local >> 1) & 1) ^ 1, &error_flag);
                int size = 0;
                for (int e = rows.next(-1); e != kNone; e = rows.next(e), ++size)
                    if (lane == 0) list[slot][size] = e;
                if (lane == 0) list_size[slot] = size;
                if (not ok) break;
                if (lane == 0) ptx::mbarrier_arrive(&list_full_bar[slot]);
            }
            position = (position + blocks) % kStages;
            // this group's first chunk of the row's t (exact when the chunks are even in number) is read before the ring has room for it
            int held = rank_chunks % 2 == 0 and (ext & 1) != group ? 1 : 0;
            float t[4][8];
            read_t(a, my_row, mine >= 0, held, t);
            ok = wait_all_lanes(&list_full_bar[slot], (local >> 1) & 1, &error_flag);
            if (not ok) break;
            const int size = list_size[slot];
            for (int i = 0; i < size and ok; ++i) {
                const int e = list[slot][i];
                for (int c = 0; c < rank_chunks; ++c, ++ext) {
                    const int s = position;
                    position = position + 1 == kStages ? 0 : position + 1;
                    if ((ext & 1) != group) continue;
                    if (mine == e and held != c) read_t(a, my_row, true, c, t);
                    // the V block has landed, so the slot is this block's
                    ok = wait_all_lanes(&v_bar[group][s], (landed >> s) & 1, &error_flag);
                    landed ^= 1u << s;
                    if (not ok) break;
                    // a row's t concerns this CTA's accumulator, a column of V both
                    if (write_t(smem_a + s * kHalf, row, mine == e, t)) poison[local % kPoisonSlots] = local + 1;
                    if (mine == e and c + 2 < rank_chunks) held = c + 2, read_t(a, my_row, true, held, t);
                    if (take_out_non_finite(smem_b + s * kHalf, a.mn_major, row)) {
                        for (int q = 0; q < 2; ++q)
                            asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(tc::map_to_cta(const_cast<const int*>(&poison[local % kPoisonSlots]), q)), "r"(local + 1) : "memory");
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbarrier_arrive_cluster(tc::map_to_cta(&ext_bar[s], 0));
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbarrier_arrive(&list_empty_bar[slot]);
        }
    } else {
        // ------------------------------------------------------------------ epilogue (both CTAs, own rows)
        const int quarter = warp & 3;
        uint8_t* buffer = smem_out + quarter * 4096;
        int local = 0;
        for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++local) {
            int m0, n0;
            origin(tile, m0, n0);
            const int acc = local & 1;
            if (not __all_sync(0xffffffffu, wait_cluster(&tmem_full_bar[acc], (local >> 1) & 1, &error_flag))) break;
            tc::fence_after_thread_sync();
            store_tile(&map_y, a, tmem + acc * 256 + (uint32_t(quarter * 32) << 16), buffer, m0 + 128 * half + quarter * 32, n0, 256,
                       poison[local % kPoisonSlots] == local + 1, lane);
            tc::fence_before_thread_sync();
            __syncwarp();
            if (lane == 0) tc::mbarrier_arrive_cluster(tc::map_to_cta(&tmem_empty_bar[acc], 0));
        }
        if (lane == 0) ptx::bulk_wait<0>();
        __syncwarp();
    }

    tc::fence_before_thread_sync();
    __syncthreads();
    tc::cluster_sync();                       // the pair's tensor memory is given back together
    if (warp == 1) {
        tc::fence_after_thread_sync();
        tc::tmem_dealloc_pair(tmem, 512);
    }
    if (threadIdx.x == 0) report(error_flag != 0, a.rows.status);
}

// ---------------------------------------------------------------------------------------- shared product + adapters, few rows
// Decode, one row tile: the time is that of reading W once. A cluster shares the contraction of block_n columns of Y, so that
// every SM pulls on W with all the shared memory it has in flight; rows of x that do not exist are not loaded (the products read
// whatever lies behind them, into accumulator rows that are never stored). The low-rank term is too small for tensor-core
// blocks of its own (a block per adapter costs about a microsecond, and every row may have another adapter): eight warps, idle
// while W streams in, compute it in fp32 for the rows their CTA owns and add it to the parts of the shared product.
//   warp 0      TMA producer     warp 1      MMA issuer
//   warps 2-9   low-rank term; warps 2-5 then send the accumulator's rows to their owners, and all eight add and store
// One tile per CTA. The wait for the kernel that computes t comes after W is under way.
// (launched with 320 threads; the bound keeps the registers at 88 or less, beside which three CTAs of lora_shrink_rows_kernel fit in each
// quarter of an SM: three warps of this kernel and six of that one)
__global__ void __launch_bounds__(736, 1)
lora_gemm_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ LoraGemmFewArgs a) {
    using namespace lora_detail;
    extern __shared__ uint8_t smem_raw[];
    constexpr int kMaxStages = 32;
    __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], done_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int error_flag;

    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) / 32, 0), lane = ptx::lane_id();
    const int cluster = a.cluster, rank = cluster > 1 ? int(blockIdx.x) % cluster : 0, tile = int(blockIdx.x) / cluster;
    const int BN = a.block_n, stages = a.num_stages, sub = a.stage_blocks;       // a stage holds `sub` K blocks
    const int n0 = tile * BN;
    const int blocks = math::ceil_div(a.k, kLoraBlockK), per = math::align(math::ceil_div(blocks, cluster), sub);
    const int kb0 = min(rank * per, blocks), kb1 = min(kb0 + per, blocks), steps = math::ceil_div(kb1 - kb0, sub);
    const uint32_t x_bytes = a.x_box_rows * kLoraBlockK * 2, w_bytes = BN * kLoraBlockK * 2;       // of one K block
    uint8_t* smem_a = align_1024(smem_raw);
    uint8_t* smem_b = smem_a + stages * sub * x_bytes;
    uint8_t* smem_part = smem_b + stages * sub * w_bytes;

    const auto load = [&](int step, int s) {
        ptx::mbarrier_arrive_expect_tx(&full_bar[s], sub * (x_bytes + w_bytes));
        for (int i = 0; i < sub; ++i) {
            // (blocks behind the contraction's end read zeros; behind this CTA's share they are not multiplied)
            const int k0 = (kb0 + step * sub + i) * kLoraBlockK;
            tc::tma_load_2d(smem_a + (s * sub + i) * x_bytes, &map_x, k0, 0, &full_bar[s]);
            uint8_t* sb = smem_b + (s * sub + i) * w_bytes;
            if (a.mn_major) for (int c = 0; c < BN / 64; ++c) tc::tma_load_2d(sb + c * 8192, &map_w, n0 + 64 * c, k0, &full_bar[s]);
            else tc::tma_load_2d(sb, &map_w, k0, n0, &full_bar[s]);
        }
    };
    if (threadIdx.x == 32) tc::prefetch_tensormap(&map_x), tc::prefetch_tensormap(&map_w);
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) ptx::mbarrier_init(&full_bar[s], 1), ptx::mbarrier_init(&empty_bar[s], 1);
        ptx::mbarrier_init(&done_bar, 1);
        ptx::fence_mbarrier_init();
        error_flag = 0;
        for (int i = 0; i < min(stages, steps); ++i) load(i, i);
    }
    if (warp == 1) tc::tmem_alloc(&tmem_slot, BN);
    tc::fence_before_thread_sync();
    __syncthreads();
    tc::fence_after_thread_sync();
    const uint32_t tmem = tmem_slot;
    tc::cluster_arrive();                     // (waited for before the first access to another CTA's shared memory)

    const int share = kLoraTileRows / cluster, units = BN / 8;                    // an item: eight columns of one row
    float low[2][8];
    if (warp == 0) {
        Ring ring;
        int issued = min(stages, steps);
        for (; issued < steps; ++issued, ring.advance(stages)) {
            if (not wait_all_lanes(&empty_bar[ring.slot], ring.phase, &error_flag)) break;
            if (elect_one()) load(issued, ring.slot);
        }
        drain(full_bar, issued, stages);      // its own copies have landed before this warp leaves, also when somebody gave up
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t idesc = tc::make_idesc(tc::kFormatBF16, kLoraTileRows, BN, false, a.mn_major);
        const uint32_t b_k = (a.mn_major ? 2048 : 32) >> 4;
        const uint64_t desc_a0 = tc::make_smem_desc(smem_a, 16, 1024), desc_b0 = tc::make_smem_desc(smem_b, a.mn_major ? 8192 : 16, 1024);
        Ring ring;
        for (int step = 0; step < steps; ++step, ring.advance(stages)) {
            wait(&full_bar[ring.slot], ring.phase, &error_flag);
            tc::fence_after_thread_sync();
            if (elect_one()) {
                for (int i = 0; i < sub and kb0 + step * sub + i < kb1; ++i) {
                    const uint64_t da = desc_a0 + uint64_t((ring.slot * sub + i) * (x_bytes >> 4)), db = desc_b0 + uint64_t((ring.slot * sub + i) * (w_bytes >> 4));
                    #pragma unroll
                    for (int k = 0; k < kLoraBlockK / 16; ++k) tc::mma_f16(tmem, da + k * 2, db + k * b_k, idesc, step > 0 or i > 0 or k > 0);
                }
                tc::commit(&empty_bar[ring.slot]);
            }
        }
        if (elect_one()) tc::commit(&done_bar);
        __syncwarp();
    }
    const int id = int(threadIdx.x) - 64;
    const auto place = [&](int item, int& row, int& c) {                         // false: not part of the result
        row = rank * share + item / units, c = item % units * 8;
        return item < share * units and row < a.rows.num_rows and n0 + c < a.n;
    };
    // low-rank term of an item in fp32, four 16-byte units of V at a time (few registers: see lora_shrink_rows_kernel)
    const auto low_rank = [&](int item, float (&v)[8]) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        int row, c;
        if (not place(item, row, c)) return;
        const int e = adapter_of(a.rows, row);
        if (e < 0) return;
        const __nv_bfloat16* base = reinterpret_cast<const __nv_bfloat16*>(a.v) + int64_t(e) * a.n * a.rows.rank;
        const float* t = a.t + int64_t(row) * a.rows.rank;
        if (a.mn_major) {
            // eight columns of the rank rows r .. r + 3
            base += n0 + c;
            #pragma unroll 1
            for (int r = 0; r < a.rows.rank; r += 4) {
                const float4 f4 = *reinterpret_cast<const float4*>(t + r);
                const float f[4] = {f4.x, f4.y, f4.z, f4.w};
                uint4 u[4];
                #pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = *reinterpret_cast<const uint4*>(base + int64_t(r + j) * a.n);
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
                    #pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float2 g = ptx::bf16x2_to_float2(w[q]);
                        v[2 * q] = fmaf(f[j], g.x, v[2 * q]), v[2 * q + 1] = fmaf(f[j], g.y, v[2 * q + 1]);
                    }
                }
            }
        } else {
            // eight rank columns of four of the columns, twice
            base += int64_t(n0 + c) * a.rows.rank;
            #pragma unroll 1
            for (int r = 0; r < a.rows.rank; r += 8) {
                float f[8];
                load8(t + r, f);
                #pragma unroll
                for (int j0 = 0; j0 < 8; j0 += 4) {
                    uint4 u[4];
                    #pragma unroll
                    for (int j = 0; j < 4; ++j) u[j] = *reinterpret_cast<const uint4*>(base + (j0 + j) * a.rows.rank + r);
                    #pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
                        #pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float2 g = ptx::bf16x2_to_float2(w[q]);
                            v[j0 + j] = fmaf(f[2 * q], g.x, v[j0 + j]), v[j0 + j] = fmaf(f[2 * q + 1], g.y, v[j0 + j]);
                        }
                    }
                }
            }
        }
    };
    if (warp >= 2) {
        // V does not depend on t: it moves into L2 while t is computed. (Read only when t was there, its round trips to memory, in
        // competition with the stream of W, took 8 us for 96 rows of 64 adapters.)
        #pragma unroll 1
        for (int item = id; item < share * units; item += 256) {
            int row, c;
            if (not place(item, row, c)) continue;
            const int e = adapter_of(a.rows, row);
            if (e < 0) continue;
            const __nv_bfloat16* base = reinterpret_cast<const __nv_bfloat16*>(a.v) + int64_t(e) * a.n * a.rows.rank;
            if (not a.mn_major)
                for (int i = 0; i < 8 * a.rows.rank; i += 64) ptx::prefetch_l2(base + int64_t(n0 + c) * a.rows.rank + i);
            else if (c % 64 == 0)
                for (int r = 0; r < a.rows.rank; ++r) ptx::prefetch_l2(base + int64_t(r) * a.n + n0 + c);
        }
        cudaGridDependencySynchronize();      // t comes from the kernel before
        #pragma unroll
        for (int i = 0; i < 2; ++i) low_rank(id + 256 * i, low[i]);
        __syncwarp();
    }
    if (warp >= 2 and warp < 6) {
        const int quarter = warp & 3, row = quarter * 32 + lane;
        wait_all_lanes(&done_bar, 0, &error_flag);
        tc::fence_after_thread_sync();
        tc::cluster_wait();
        if (quarter * 32 < a.rows.num_rows)
            send_part(tc::map_to_cta(smem_part + (rank * share + row % share) * (BN * 4), row / share), tmem + (uint32_t(quarter * 32) << 16), BN, row,
                      row < a.rows.num_rows);
        tc::fence_before_thread_sync();
        __syncwarp();
    } else {
        tc::cluster_wait();
    }
    tc::cluster_sync();                       // all parts have arrived; nobody touches another CTA's shared memory after this
    if (warp >= 2) {
        for (int first = id; first < share * units; first += 512) {
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                int row, c;
                if (first != id) low_rank(first + 256 * i, low[i]);
                if (not place(first + 256 * i, row, c)) continue;
                float v[8] = {};
                add_parts(v, smem_part, share * BN * 4, cluster, (row % share) * BN * 4, c, row);
                #pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += low[i][j];
                store8(reinterpret_cast<__nv_bfloat16*>(a.y) + int64_t(row) * a.n + n0 + c, v);
            }
        }
    }
    tc::fence_before_thread_sync();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_thread_sync();
        tc::tmem_dealloc(tmem, BN);
    }
    if (threadIdx.x == 0) report(error_flag != 0, a.rows.status);
}

// ---------------------------------------------------------------------------------------- weight gradients
// A cluster owns (adapter, 256 columns of X); its CTAs take the adapter's row tiles in turn and add their sums through
// distributed shared memory in rank order. X is the A operand (its columns are the M of the product), t the B operand, written
// into shared memory as hi and lo side by side: one product gives both sums, which are added at the end. Row tiles in which the adapter does not occur are never read.
//   warp 0      TMA producer     warp 1      MMA issuer
//   warps 2-9   writers of t, two groups that take the blocks in turn; warps 2-5 read the accumulator
// A block of 64 tokens is little work for the tensor cores, so the writers set the pace: each asks for the index two blocks
// ahead and for t one block ahead, into registers of its own for every other block. Measured with 4099 rows of 4 adapters in runs,
// 7168 columns: 22 / 25 / 69 us at rank 16 / 32 / 128 (one register set, copied from block to block: 28 / 32 / 66 us; one group that
// read both when it needed them: 1.4 us per block). Rows in another order cost each adapter the row tiles in which it occurs.
constexpr int kLoraWgradColumns = 256;

// kUnits: units of eight rank columns per writer thread (two threads share a row)
template <int kUnits>
__global__ void __launch_bounds__(320, 1)
lora_wgrad_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LoraWgradArgs a) {
    using namespace lora_detail;
    extern __shared__ uint8_t smem_raw[];
    constexpr int kMaxStages = 4, kM = kLoraWgradColumns;
    constexpr uint32_t kXBytes = kM * kLoraBlockK * 2;          // 64 tokens x 256 columns, blocks of 64 columns
    __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], ext_bar[kMaxStages], done_bar;
    __shared__ uint32_t tmem_slot, tile_bits[kLoraMaxTileWords];
    __shared__ volatile int error_flag;

    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) / 32, 0), lane = ptx::lane_id();
    const int cluster = a.cluster, rank = blockIdx.x % cluster, item = blockIdx.x / cluster;
    const int m_tile = item % a.m_tiles, e = item / a.m_tiles, m0 = m_tile * kM;
    // columns of t: hi in [0, half), lo in [half, 2 * half); those beyond the rank hold whatever is there, and so do the columns of
    // the accumulator that they make, which nobody reads
    const int half = a.rows.rank <= 32 ? 32 : math::align(a.rows.rank, 64), stages = a.num_stages;
    const int words = math::ceil_div(a.row_tiles, 32), pitch = math::align(a.rows.rank, 16) + 4;      // floats per column of X, staged
    uint8_t* smem = align_1024(smem_raw);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) ptx::mbarrier_init(&full_bar[s], 1), ptx::mbarrier_init(&empty_bar[s], 1), ptx::mbarrier_init(&ext_bar[s], 4);
        ptx::mbarrier_init(&done_bar, 1);
        ptx::fence_mbarrier_init();
        error_flag = 0;
        tc::prefetch_tensormap(&map_x);
    }
    for (int w = warp; w < words; w += 10) {
        const int tile = w * 32 + lane;
        const unsigned bits = __ballot_sync(0xffffffffu, tile < a.row_tiles and a.presence[int64_t(tile) * a.rows.num_adapters + e] != 0);
        if (lane == 0) tile_bits[w] = bits;
    }
    uint32_t columns = 32;
    while (columns < uint32_t(4 * half)) columns *= 2;
    if (warp == 1) tc::tmem_alloc(&tmem_slot, columns);
    tc::fence_before_thread_sync();
    __syncthreads();
    tc::fence_after_thread_sync();
    const uint32_t tmem = tmem_slot;

    // every role walks the blocks of 64 tokens in the same order; `body(token0)` returns false to give up
    const auto walk = [&](auto body) {
        int turn = 0;
        for (int w = 0; w < words; ++w)
            for (unsigned bits = tile_bits[w]; bits != 0; bits &= bits - 1) {
                const int token = (w * 32 + __ffs(int(bits)) - 1) * kLoraTileRows;
                for (int half = 0; half < 2 and token + half * kLoraBlockK < a.rows.num_rows; ++half, ++turn)
                    if (turn % cluster == rank and not body(token + half * kLoraBlockK)) return;
            }
    };

    int count = 0;                            // blocks of this CTA
    if (warp == 0) {
        Ring ring;
        walk([&](int token) {
            if (not wait_all_lanes(&empty_bar[ring.slot], ring.phase ^ 1, &error_flag)) return false;
            if (elect_one()) {
                ptx::mbarrier_arrive_expect_tx(&full_bar[ring.slot], kXBytes);
                uint8_t* stage = smem + size_t(ring.slot) * a.stage_bytes;
                #pragma unroll
                for (int i = 0; i < kM / 64; ++i) tc::tma_load_2d(stage + i * 8192, &map_x, m0 + 64 * i, token, &full_bar[ring.slot]);
            }
            ++count, ring.advance(stages);
            return true;
        });
        drain(full_bar, count, stages);       // its own copies have landed before this warp leaves, also when somebody gave up
    } else if (warp == 1) {
        const uint32_t idesc = tc::make_idesc(tc::kFormatBF16, 128, 2 * half, true, true);
        const uint64_t desc_x = tc::make_smem_desc(smem, 8192, 1024), desc_t = tc::make_smem_desc(smem + kXBytes, 8192, 1024);
        Ring ring;
        walk([&](int) {
            wait(&full_bar[ring.slot], ring.phase, &error_flag);
            wait(&ext_bar[ring.slot], ring.phase, &error_flag);
            tc::fence_after_thread_sync();
            if (elect_one()) {
                const uint64_t step = uint64_t(ring.slot) * (a.stage_bytes >> 4);
                #pragma unroll
                for (int k = 0; k < kLoraBlockK / 16; ++k) {
                    #pragma unroll
                    for (int m = 0; m < 2; ++m)                 // 128 columns of X each, 16 KB apart
                        tc::mma_f16(tmem + m * 2 * half, desc_x + step + m * 1024 + k * 128, desc_t + step + k * 128, idesc, count > 0 or k > 0);
                }
                tc::commit(&empty_bar[ring.slot]);
            }
            ++count, ring.advance(stages);
            return true;
        });
        if (elect_one()) tc::commit(&done_bar);
    } else {
        // ------------------------------------------------------------------ writers of the B operand, then the epilogue
        const int id = (threadIdx.x - 64) & 127, group = (warp - 2) / 4, line = id & 63, side = id >> 6;
        // a block's index is asked for in one step, its t in the next, and it is written in the one after that
        int first = -1, first_turn = 0, first32 = -1;           // block whose index has been asked for: first token, number, index as read
        int64_t first64 = -1;
        int second = -1, second_turn = 0, turn = 0;             // block whose t has been asked for
        bool second_mine = false, odd = false;
        float t_even[kUnits][8], t_odd[kUnits][8];              // of alternate blocks: a copy would wait for the read
        const auto write = [&](const float (&values)[kUnits][8]) {
            const int s = second_turn % stages, phase = (second_turn / stages) & 1;
            uint8_t* stage = smem + size_t(s) * a.stage_bytes;
            if (not wait_all_lanes(&empty_bar[s], phase ^ 1, &error_flag)) return false;
            const auto place = [&](int column) {                // 16-byte unit of this row's line in its block of 64 columns
                return reinterpret_cast<uint4*>(stage + kXBytes + (column / 64) * 8192 + line * 128 + (((column % 64 / 8) ^ (line & 7)) << 4));
            };
            #pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = 8 * (2 * i + side);
                if (r < a.rows.rank) split8<false>(values[i], *place(r), *place(half + r));
            }
            // rows of other requests in this block: zeros instead of whatever they hold (0 * inf would be NaN)
            const bool foreign = not second_mine and second + line < a.rows.num_rows;
            if (__any_sync(0xffffffffu, foreign)) {
                if (not wait_all_lanes(&full_bar[s], phase, &error_flag)) return false;
                if (foreign)
                    for (int i = side; i < kM / 64; i += 2)
                        for (int u = 0; u < 8; ++u) *reinterpret_cast<uint4*>(stage + i * 8192 + line * 128 + u * 16) = make_uint4(0, 0, 0, 0);
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbarrier_arrive(&ext_bar[s]);
            return true;
        };
        // one step of the pipeline: `token` enters (-1: none), what leaves it is written
        const auto advance = [&](int token, int token_turn, const float (&now)[kUnits][8], float (&next)[kUnits][8]) {
            // (compared with the adapter in the next step: a comparison here would wait for the read)
            int new32 = -1;
            int64_t new64 = -1;
            if (token >= 0 and token + line < a.rows.num_rows) {
                if (a.rows.idx64) new64 = reinterpret_cast<const int64_t*>(a.rows.idx)[token + line];
                else new32 = reinterpret_cast<const int*>(a.rows.idx)[token + line];
            }
            const bool mine = a.rows.idx64 ? first64 == e : first32 == e;
            #pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int u = 2 * i + side;
                #pragma unroll
                for (int j = 0; j < 8; ++j) next[i][j] = 0.0f;
                if (mine and 8 * u < a.rows.rank) load8(a.t + int64_t(first + line) * a.rows.rank + 8 * u, next[i]);
            }
            if (second >= 0 and not write(now)) return false;
            second = first, second_mine = mine, second_turn = first_turn;
            first = token, first32 = new32, first64 = new64, first_turn = token_turn;
            return true;
        };
        const auto step = [&](int token, int token_turn) {
            odd = not odd;
            return odd ? advance(token, token_turn, t_even, t_odd) : advance(token, token_turn, t_odd, t_even);
        };
        walk([&](int token) {
            const int this_turn = turn++;
            count = turn;
            return this_turn % 2 != group or step(token, this_turn);
        });
        if (step(-1, 0)) step(-1, 0);
        if (warp < 6) {
            wait_all_lanes(&done_bar, 0, &error_flag);
            tc::fence_after_thread_sync();
            const int quarter = warp & 3;
            float* part = reinterpret_cast<float*>(smem);
            // an infinity or NaN of X shows in hi's products as in those of t itself, lo's products with it have another sign or are NaN
            const auto sum = [](uint32_t hi, uint32_t lo) {
                const float h = __uint_as_float(hi);
                return isfinite(h) ? h + __uint_as_float(lo) : h;
            };
            for (int m = 0; m < 2; ++m) {
                float* out = part + (m * 128 + quarter * 32 + lane) * pitch;
                for (int c = 0; c < a.rows.rank; c += 16) {
                    uint32_t r[16], q[16];
                    const uint32_t at = tmem + (uint32_t(quarter * 32) << 16) + m * 2 * half + c;
                    tc::tmem_ld_32x16(at, r);
                    tc::tmem_ld_32x16(at + half, q);
                    tc::wait_ld();
                    #pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (count > 0) v = make_float4(sum(r[i], q[i]), sum(r[i + 1], q[i + 1]), sum(r[i + 2], q[i + 2]), sum(r[i + 3], q[i + 3]));
                        *reinterpret_cast<float4*>(out + c + i) = v;
                    }
                }
            }
            tc::fence_before_thread_sync();
        }
    }
    __syncthreads();
    if (cluster > 1) tc::cluster_sync();
    bool any = false;
    for (int w = 0; w < words; ++w) any = any or tile_bits[w] != 0;
    if (any or not a.accumulate) {
        const float* part = reinterpret_cast<const float*>(smem);
        const int share = kM / cluster, first = rank * share, units = a.rows.rank / 4;
        for (int i = threadIdx.x; i < share * units; i += 320) {
            // an item is four rank columns of one column of X; neighbouring threads write neighbouring addresses in either layout
            const int m = first + (a.rank_major ? i % share : i / units), r = (a.rank_major ? i / share : i % units) * 4;
            if (m0 + m >= a.m) continue;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            const float* line = part + m * pitch + r;
            for (int q = 0; q < cluster; ++q) {
                const float4 v = cluster > 1 ? ld_cluster_v4(tc::map_to_cta(line, q)) : *reinterpret_cast<const float4*>(line);
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
            if (a.rank_major) {
                const float v[4] = {sum.x, sum.y, sum.z, sum.w};
                const int64_t at = (int64_t(e) * a.rows.rank + r) * a.m + m0 + m;
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (a.out_fp32) {
                        float* d = reinterpret_cast<float*>(a.d) + at + int64_t(j) * a.m;
                        *d = a.accumulate ? *d + v[j] : v[j];
                    } else {
                        reinterpret_cast<__nv_bfloat16*>(a.d)[at + int64_t(j) * a.m] = __float2bfloat16_rn(v[j]);
                    }
                }
            } else {
                const int64_t at = (int64_t(e) * a.m + m0 + m) * a.rows.rank + r;
                if (a.out_fp32) {
                    // (a buffer of the caller's may lie on any 4-byte boundary)
                    float* d = reinterpret_cast<float*>(a.d) + at;
                    if (a.accumulate) sum.x += d[0], sum.y += d[1], sum.z += d[2], sum.w += d[3];
                    if (reinterpret_cast<uintptr_t>(d) % 16 == 0) *reinterpret_cast<float4*>(d) = sum;
                    else d[0] = sum.x, d[1] = sum.y, d[2] = sum.z, d[3] = sum.w;
                } else {
                    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.d) + at) =
                        make_uint2(ptx::float2_to_bf16x2(sum.x, sum.y), ptx::float2_to_bf16x2(sum.z, sum.w));
                }
            }
        }
    }
    if (cluster > 1) tc::cluster_sync();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_thread_sync();
        tc::tmem_dealloc(tmem, columns);
    }
    if (threadIdx.x == 0) report(error_flag != 0, a.rows.status);
}

}  // namespace deep_ep::kernels
