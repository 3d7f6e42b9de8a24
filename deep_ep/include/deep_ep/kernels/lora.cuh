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
// Zeros do not hide infinities or NaN (0 * inf = NaN). lora_gemm therefore looks for them in the adapter's block whenever a
// tile holds other rows too, takes them out of the tensor cores' operand, and adds their products to the owner's rows
// separately; lora_wgrad overwrites the rows of other requests with zeros. One request cannot poison another.
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

// The adapters of a tile's 128 rows, four rows per lane: enumerated in ascending order by minimum search, which needs no
// list, no sort and no other kernel. Every role that needs the order walks it on its own.
struct TileAdapters {
    int id[4];
    bool inside[4];

    EP_DEVICE void load(const LoraRows& r, int m0, int lane) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = m0 + lane + 32 * i;
            inside[i] = row < r.num_rows;
            id[i] = adapter_of(r, row);
        }
    }
    EP_DEVICE int next(int last) const {
        unsigned best = kNone;
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            if (id[i] > last) best = min(best, static_cast<unsigned>(id[i]));
        return static_cast<int>(__reduce_min_sync(0xffffffffu, best));
    }
    // some row of the batch in this tile has another adapter (or none) than `e`
    EP_DEVICE bool others_than(int e) const {
        bool other = false;
        #pragma unroll
        for (int i = 0; i < 4; ++i) other = other or (inside[i] and id[i] != e);
        return __any_sync(0xffffffffu, other);
    }
};

EP_DEVICE bool has_non_finite(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    bool bad = false;
    #pragma unroll
    for (int i = 0; i < 4; ++i) bad = bad or (w[i] & 0x7f80u) == 0x7f80u or (w[i] & 0x7f800000u) == 0x7f800000u;
    return bad;
}

// v = hi + lo with both bf16 (an infinite or NaN v has no rest)
EP_DEVICE void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = ptx::float2_to_bf16x2(a, b);
    const float2 h = ptx::bf16x2_to_float2(hi);
    const float ra = a - h.x, rb = b - h.y;
    lo = ptx::float2_to_bf16x2(isfinite(ra) ? ra : 0.0f, isfinite(rb) ? rb : 0.0f);
}
// eight values -> one 16-byte unit each of hi and lo
EP_DEVICE void split8(const float (&v)[8], uint4& hi, uint4& lo) {
    uint32_t h[4], l[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) split2(v[2 * i], v[2 * i + 1], h[i], l[i]);
    hi = make_uint4(h[0], h[1], h[2], h[3]), lo = make_uint4(l[0], l[1], l[2], l[3]);
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

    cudaTriggerProgrammaticLaunchCompletion();
    const int warp = threadIdx.x / 32, lane = ptx::lane_id();
    const int cluster = a.cluster, rank = blockIdx.x % cluster;
    const int chunk = (blockIdx.x / cluster) % a.num_chunks, tile = blockIdx.x / cluster / a.num_chunks;
    const int m0 = tile * kLoraTileRows;
    // columns of the accumulator per adapter: the rank, padded (by zeros that the TMA fills in) to what the operand's layout has
    const int rp = math::align(a.rows.rank, a.mn_major ? 64 : 16), stages = a.num_stages;
    uint8_t* smem = align_1024(smem_raw);
    constexpr uint32_t kXBytes = kLoraTileRows * kLoraBlockK * 2;
    const uint32_t slot_bytes = rp * 128u;    // one adapter's block of a stage

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) ptx::mbarrier_init(&full_bar[s], 1), ptx::mbarrier_init(&empty_bar[s], 1);
        ptx::mbarrier_init(&done_bar, 1);
        ptx::fence_mbarrier_init();
        error_flag = 0;
        tc::prefetch_tensormap(&map_x), tc::prefetch_tensormap(&map_a);
    }
    if (warp == 0) {
        // this chunk's adapters
        TileAdapters rows;
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
        if (lane == 0) {
            int issued = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                const int s = issued % stages;
                if (not ptx::mbarrier_wait(&empty_bar[s], ((issued / stages) & 1) ^ 1)) { error_flag = 1; break; }
                uint8_t* stage = smem + size_t(s) * a.stage_bytes;
                ptx::mbarrier_arrive_expect_tx(&full_bar[s], kXBytes + n * slot_bytes);
                tc::tma_load_2d(stage, &map_x, kb * kLoraBlockK, m0, &full_bar[s]);
                for (int j = 0; j < n; ++j) {
                    uint8_t* dst = stage + kXBytes + j * slot_bytes;
                    if (a.mn_major) {
                        for (int c = 0; c * 64 < rp; ++c) tc::tma_load_3d(dst + c * 8192, &map_a, c * 64, kb * kLoraBlockK, list[j], &full_bar[s]);
                    } else {
                        tc::tma_load_3d(dst, &map_a, kb * kLoraBlockK, 0, list[j], &full_bar[s]);
                    }
                }
            }
            // its own copies have landed before this thread leaves, also when somebody gave up
            for (int i = max(0, issued - stages); i < issued; ++i) ptx::mbarrier_wait(&full_bar[i % stages], (i / stages) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = tc::make_idesc(tc::kFormatBF16, kLoraTileRows, rp, false, a.mn_major);
            const uint32_t b_lead = a.mn_major ? 8192 : 16, b_k = (a.mn_major ? 2048 : 32) >> 4;
            const uint64_t desc_x = tc::make_smem_desc(smem, 16, 1024), desc_a = tc::make_smem_desc(smem + kXBytes, b_lead, 1024);
            for (int kb = kb0; kb < kb1; ++kb) {
                const int i = kb - kb0, s = i % stages;
                if (error_flag or not ptx::mbarrier_wait(&full_bar[s], (i / stages) & 1)) { error_flag = 1; break; }
                tc::fence_after_thread_sync();
                const uint64_t step = uint64_t(s) * (a.stage_bytes >> 4);
                for (int j = 0; j < n; ++j) {
                    #pragma unroll
                    for (int k = 0; k < kLoraBlockK / 16; ++k)
                        tc::mma_f16(tmem + j * rp, desc_x + step + k * 2, desc_a + step + uint64_t(j) * (slot_bytes >> 4) + k * b_k, idesc, i > 0 or k > 0);
                }
                tc::commit(&empty_bar[s]);
            }
            tc::commit(&done_bar);
        }
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
        if (not ptx::mbarrier_wait(&done_bar, 0)) error_flag = 1;
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

// ---------------------------------------------------------------------------------------- shared product + adapters
// Tiles of 128 rows x BN columns. Many tiles: persistent CTAs, two accumulators in tensor memory, so that the stores of one tile
// overlap the products of the next. Few tiles (decode): a cluster shares the tile's contraction, so that all SMs pull on W,
// and adds its parts through distributed shared memory in rank order.
//   warp 0      TMA producer: K blocks of x and W, then the V blocks of the tile's adapters
//   warp 1      MMA issuer
//   warps 2-5   epilogue
//   warps 6-9   writers: the A operand of the adapters' K blocks (t as bf16 hi | lo, zeros in the rows of others)
template <int BN>
__global__ void __launch_bounds__(320, 1)
lora_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap map_y, const __grid_constant__ LoraGemmArgs a) {
    using namespace lora_detail;
    extern __shared__ uint8_t smem_raw[];
    constexpr int kStages = BN == 256 ? 4 : 6, kGroupM = 16;
    constexpr uint32_t kABytes = kLoraTileRows * kLoraBlockK * 2, kBBytes = BN * kLoraBlockK * 2;
    constexpr int kPoisonSlots = 8;           // more tiles than the ring can run ahead
    __shared__ uint64_t full_bar[kStages], empty_bar[kStages], grant_bar[kStages], ext_bar[kStages], tmem_full_bar[2], tmem_empty_bar[2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int error_flag, poison[kPoisonSlots];

    const int warp = threadIdx.x / 32, lane = ptx::lane_id();
    const int cluster = a.cluster, rank = cluster > 1 ? int(blockIdx.x) % cluster : 0;
    const int num_tiles = a.m_tiles * a.n_tiles;
    const int first_tile = int(blockIdx.x) / cluster, tile_step = int(gridDim.x) / cluster;
    uint8_t* smem_a = align_1024(smem_raw);
    uint8_t* smem_b = smem_a + kStages * kABytes;
    uint8_t* smem_out = smem_b + kStages * kBBytes;            // 4 x 4 KB, one chunk of 32 rows x 64 columns per epilogue warp

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s)
            ptx::mbarrier_init(&full_bar[s], 1), ptx::mbarrier_init(&empty_bar[s], 1), ptx::mbarrier_init(&grant_bar[s], 1), ptx::mbarrier_init(&ext_bar[s], 4);
        for (int i = 0; i < 2; ++i) ptx::mbarrier_init(&tmem_full_bar[i], 1), ptx::mbarrier_init(&tmem_empty_bar[i], 4);
        ptx::fence_mbarrier_init();
        error_flag = 0;
        for (int i = 0; i < kPoisonSlots; ++i) poison[i] = 0;
        tc::prefetch_tensormap(&map_x), tc::prefetch_tensormap(&map_w), tc::prefetch_tensormap(&map_v), tc::prefetch_tensormap(&map_y);
    }
    if (warp == 1) tc::tmem_alloc(&tmem_slot, 2 * BN);
    tc::fence_before_thread_sync();
    __syncthreads();
    tc::fence_after_thread_sync();
    const uint32_t tmem = tmem_slot;

    const int blocks = math::ceil_div(a.k, kLoraBlockK), per = math::ceil_div(blocks, cluster);
    const int kb0 = min(rank * per, blocks), kb1 = min(kb0 + per, blocks);        // never empty, see the launcher
    const int rank_chunks = math::ceil_div(a.rows.rank, 32);                      // 32 rank columns (hi and lo) per K block

    // tile -> origin; groups of 16 row tiles run through all columns, so that their rows of x and all of W stay in L2
    const auto origin = [&](int tile, int& m0, int& n0) {
        const int group = tile / (kGroupM * a.n_tiles), first_m = group * kGroupM, gm = min(kGroupM, a.m_tiles - first_m);
        const int local = tile - group * kGroupM * a.n_tiles;
        m0 = (first_m + local % gm) * kLoraTileRows, n0 = local / gm * BN;
    };

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        unsigned it = 0;
        bool ok = true;
        for (int tile = first_tile; tile < num_tiles and ok; tile += tile_step) {
            int m0, n0;
            origin(tile, m0, n0);
            TileAdapters rows;
            rows.load(a.rows, m0, lane);
            if (lane == 0) {
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const unsigned s = it % kStages;
                    if (error_flag or not ptx::mbarrier_wait(&empty_bar[s], ((it / kStages) & 1) ^ 1)) { error_flag = 1, ok = false; break; }
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
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0), it = __shfl_sync(0xffffffffu, it, 0);
            int turn = 0;
            for (int e = rows.next(-1); e != kNone and ok; e = rows.next(e), ++turn) {
                if (turn % cluster != rank) continue;
                for (int c = 0; c < rank_chunks and ok; ++c) {
                    const unsigned s = it % kStages;
                    if (lane == 0) {
                        if (error_flag or not ptx::mbarrier_wait(&empty_bar[s], ((it / kStages) & 1) ^ 1)) {
                            error_flag = 1, ok = false;
                        } else {
                            ptx::mbarrier_arrive(&grant_bar[s]);            // the writers may fill the A slot
                            ptx::mbarrier_arrive_expect_tx(&full_bar[s], kBBytes);
                            uint8_t* sb = smem_b + s * kBBytes;
                            if (a.mn_major) {
                                #pragma unroll
                                for (int i = 0; i < BN / 64; ++i) tc::tma_load_3d(sb + i * 8192, &map_v, n0 + 64 * i, 32 * c, e, &full_bar[s]);
                            } else {
                                #pragma unroll
                                for (int i = 0; i < BN / 128; ++i) tc::tma_load_3d(sb + i * 16384, &map_v, 32 * c, n0 + 128 * i, e, &full_bar[s]);
                            }
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    it += ok;
                }
            }
        }
        // its own copies have landed before this warp leaves, also when somebody gave up
        if (lane == 0)
            for (unsigned i = it > kStages ? it - kStages : 0; i < it; ++i) ptx::mbarrier_wait(&full_bar[i % kStages], (i / kStages) & 1);
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        const uint32_t idesc = tc::make_idesc(tc::kFormatBF16, kLoraTileRows, BN, false, a.mn_major);
        const uint32_t b_lead = a.mn_major ? 8192 : 16, b_k = (a.mn_major ? 2048 : 32) >> 4;
        const uint64_t desc_a0 = tc::make_smem_desc(smem_a, 16, 1024), desc_b0 = tc::make_smem_desc(smem_b, b_lead, 1024);
        unsigned it = 0, ext_phase = 0;
        int local = 0;
        bool ok = true;
        for (int tile = first_tile; tile < num_tiles and ok; tile += tile_step, ++local) {
            int m0, n0;
            origin(tile, m0, n0);
            TileAdapters rows;
            rows.load(a.rows, m0, lane);
            const int acc = local & 1;
            const uint32_t d = tmem + acc * BN;
            if (lane == 0) {
                if (not ptx::mbarrier_wait(&tmem_empty_bar[acc], ((local >> 1) & 1) ^ 1)) error_flag = 1, ok = false;
                tc::fence_after_thread_sync();
                for (int kb = kb0; kb < kb1 and ok; ++kb, ++it) {
                    const unsigned s = it % kStages;
                    if (error_flag or not ptx::mbarrier_wait(&full_bar[s], (it / kStages) & 1)) { error_flag = 1, ok = false; break; }
                    tc::fence_after_thread_sync();
                    const uint64_t da = desc_a0 + uint64_t(s * (kABytes >> 4)), db = desc_b0 + uint64_t(s * (kBBytes >> 4));
                    #pragma unroll
                    for (int k = 0; k < kLoraBlockK / 16; ++k) tc::mma_f16(d, da + k * 2, db + k * b_k, idesc, kb > kb0 or k > 0);
                    tc::commit(&empty_bar[s]);
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0), it = __shfl_sync(0xffffffffu, it, 0);
            int turn = 0;
            for (int e = rows.next(-1); e != kNone and ok; e = rows.next(e), ++turn) {
                if (turn % cluster != rank) continue;
                for (int c = 0; c < rank_chunks and ok; ++c, ++it) {
                    const unsigned s = it % kStages;
                    if (lane == 0) {
                        if (error_flag or not ptx::mbarrier_wait(&full_bar[s], (it / kStages) & 1) or
                            not ptx::mbarrier_wait(&ext_bar[s], (ext_phase >> s) & 1)) {
                            error_flag = 1, ok = false;
                        } else {
                            tc::fence_after_thread_sync();
                            const uint64_t da = desc_a0 + uint64_t(s * (kABytes >> 4)), db = desc_b0 + uint64_t(s * (kBBytes >> 4));
                            for (int k = 0; k < 2 and 32 * c + 16 * k < a.rows.rank; ++k) {
                                tc::mma_f16(d, da + k * 2, db + k * b_k, idesc, true);             // hi
                                tc::mma_f16(d, da + 4 + k * 2, db + k * b_k, idesc, true);         // lo
                            }
                            tc::commit(&empty_bar[s]);
                        }
                    }
                    ext_phase ^= 1u << s;
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                }
            }
            if (lane == 0 and ok) tc::commit(&tmem_full_bar[acc]);
        }
    } else if (warp >= 6) {
        // ------------------------------------------------------------------ writers of the adapters' A operand
        cudaGridDependencySynchronize();      // t comes from the kernel before, which this one does not wait for until here
        const int row = threadIdx.x - 192;
        // These warps do not follow the ring through the K blocks of x, so they cannot tell from a slot's own barriers (which
        // show a phase's parity only) whether it is free for THIS block: the producer, which can, grants it.
        unsigned it = 0, granted = 0;
        int local = 0;
        bool ok = true;
        for (int tile = first_tile; tile < num_tiles and ok; tile += tile_step, ++local) {
            int m0, n0;
            origin(tile, m0, n0);
            TileAdapters rows;
            rows.load(a.rows, m0, lane);
            const int mine = adapter_of(a.rows, m0 + row);
            it += kb1 - kb0;
            int turn = 0;
            for (int e = rows.next(-1); e != kNone and ok; e = rows.next(e), ++turn) {
                if (turn % cluster != rank) continue;
                const bool shared_tile = rows.others_than(e);
                for (int c = 0; c < rank_chunks and ok; ++c, ++it) {
                    const unsigned s = it % kStages, phase = (it / kStages) & 1;
                    float v[4][8];
                    #pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const bool there = mine == e and 32 * c + 8 * u < a.rows.rank;
                        if (there) load8(a.t + int64_t(m0 + row) * a.rows.rank + 32 * c + 8 * u, v[u]);
                        #pragma unroll
                        for (int j = 0; j < 8; ++j) v[u][j] = there ? v[u][j] : 0.0f;
                    }
                    ok = ptx::mbarrier_wait(&grant_bar[s], (granted >> s) & 1);
                    granted ^= 1u << s;
                    ok = __all_sync(0xffffffffu, ok);
                    if (not ok) { error_flag = 1; break; }
                    uint8_t* line = smem_a + s * kABytes + row * 128;
                    #pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint4 hi, lo;
                        split8(v[u], hi, lo);
                        // 16-byte unit u of row r sits at unit u ^ (r % 8) of its 128-byte line
                        *reinterpret_cast<uint4*>(line + ((u ^ (row & 7)) << 4)) = hi;
                        *reinterpret_cast<uint4*>(line + (((4 + u) ^ (row & 7)) << 4)) = lo;
                    }
                    if (shared_tile) {
                        // infinities and NaN of this adapter must not meet the zeros of other rows
                        ok = ok and ptx::mbarrier_wait(&full_bar[s], phase);
                        uint8_t* sb = smem_b + s * kBBytes;
                        // the part of the block that the products read: 32 columns of BN lines, or 32 lines of each 64-column block
                        const auto look = [&](uint8_t* at) {
                            uint4* unit = reinterpret_cast<uint4*>(at);
                            if (has_non_finite(*unit)) *unit = make_uint4(0, 0, 0, 0), poison[local % kPoisonSlots] = local + 1;
                        };
                        if (a.mn_major) {
                            for (int i = row; i < BN / 64 * 32 * 8; i += 128) look(sb + (i / 256) * 8192 + (i % 256) * 16);
                        } else {
                            for (int i = row; i < BN * 4; i += 128) look(sb + (i / 4) * 128 + (((i % 4) ^ ((i / 4) & 7)) << 4));
                        }
                    }
                    ptx::fence_proxy_async_smem();
                    ok = __all_sync(0xffffffffu, ok);
                    if (not ok) { error_flag = 1; break; }
                    if (lane == 0) ptx::mbarrier_arrive(&ext_bar[s]);
                }
            }
            ok = ok and not __any_sync(0xffffffffu, error_flag != 0);
        }
    }

    // products of an adapter's infinities and NaN (whole units of eight V elements that hold one) with this row's t
    const auto poisoned = [&](int row, int n) {
        const int e = adapter_of(a.rows, row);
        if (e < 0) return 0.0f;
        const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(a.v) + int64_t(e) * a.n * a.rows.rank;
        const float* t = a.t + int64_t(row) * a.rows.rank;
        float sum = 0.0f;
        if (a.mn_major) {
            for (int r = 0; r < a.rows.rank; ++r) {
                const __nv_bfloat16* unit = v + int64_t(r) * a.n + (n & ~7);
                if (has_non_finite(*reinterpret_cast<const uint4*>(unit))) sum += t[r] * __bfloat162float(unit[n & 7]);
            }
        } else {
            for (int r = 0; r < a.rows.rank; r += 8) {
                const __nv_bfloat16* unit = v + int64_t(n) * a.rows.rank + r;
                if (has_non_finite(*reinterpret_cast<const uint4*>(unit)))
                    for (int j = 0; j < 8; ++j) sum += t[r + j] * __bfloat162float(unit[j]);
            }
        }
        return sum;
    };

    if (warp >= 2 and warp < 6) {
        // ------------------------------------------------------------------ epilogue
        const int quarter = warp & 3, row = quarter * 32 + lane;
        uint8_t* buffer = smem_out + quarter * 4096;
        int local = 0;
        for (int tile = first_tile; tile < num_tiles; tile += tile_step, ++local) {
            int m0, n0;
            origin(tile, m0, n0);
            const int acc = local & 1;
            if (error_flag or not ptx::mbarrier_wait(&tmem_full_bar[acc], (local >> 1) & 1)) { error_flag = 1; break; }
            tc::fence_after_thread_sync();
            const uint32_t taddr = tmem + acc * BN + (uint32_t(quarter * 32) << 16);
            if (cluster > 1) {
                // fp32 parts to this CTA's shared memory (the ring is idle: every product that read it has completed)
                float* part = reinterpret_cast<float*>(smem_a) + row * (BN + 4);
                for (int c = 0; c < BN; c += 32) {
                    uint32_t r[32];
                    tc::tmem_ld_32x32(taddr + c, r);
                    tc::wait_ld();
                    #pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4*>(part + c + 4 * i) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                }
            } else {
                const bool fix = poison[local % kPoisonSlots] == local + 1;          // rare; the same for the whole warp
                if (fix) cudaGridDependencySynchronize();
                for (int c = 0; c < BN; c += 64) {
                    uint8_t* line = buffer + lane * 128;
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
                        for (int j = 0; j < 64; ++j) {
                            const uint32_t r = tc::tmem_ld_32x1(taddr + c + j);
                            tc::wait_ld();
                            float v = __uint_as_float(r);
                            if (m0 + row < a.rows.num_rows and n0 + c + j < a.n) v += poisoned(m0 + row, n0 + c + j);
                            __syncwarp();
                            *reinterpret_cast<__nv_bfloat16*>(line + (((j / 8) ^ (lane & 7)) << 4) + (j % 8) * 2) = __float2bfloat16_rn(v);
                        }
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    // rows and columns beyond the matrix are cut off by the store itself
                    if (lane == 0 and m0 + quarter * 32 < a.rows.num_rows and n0 + c < a.n) {
                        tc::tma_store_2d(&map_y, n0 + c, m0 + quarter * 32, buffer);
                        ptx::bulk_commit();
                    }
                }
            }
            tc::fence_before_thread_sync();
            __syncwarp();
            if (lane == 0) ptx::mbarrier_arrive(&tmem_empty_bar[acc]);
        }
        if (lane == 0) ptx::bulk_wait<0>();
        __syncwarp();
    }

    if (cluster > 1) {
        __syncwarp();
        tc::cluster_sync();
        int m0, n0;
        origin(first_tile, m0, n0);
        bool fix = false;
        for (int q = 0; q < cluster; ++q) fix = fix or ld_cluster_int(tc::map_to_cta(const_cast<const int*>(&poison[0]), q)) != 0;
        if (fix) cudaGridDependencySynchronize();
        const int share = kLoraTileRows / cluster;
        const float* part = reinterpret_cast<const float*>(smem_a);
        for (int item = threadIdx.x; item < share * (BN / 8); item += 320) {
            const int row = rank * share + item / (BN / 8), c = item % (BN / 8) * 8;
            if (m0 + row >= a.rows.num_rows or n0 + c >= a.n) continue;
            float v[8] = {};
            for (int q = 0; q < cluster; ++q) {
                const uint32_t at = tc::map_to_cta(part + row * (BN + 4) + c, q);
                const float4 x = ld_cluster_v4(at), y = ld_cluster_v4(at + 16);
                v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
            }
            if (fix) {
                for (int j = 0; j < 8; ++j) v[j] += poisoned(m0 + row, n0 + c + j);
            }
            uint4 packed = make_uint4(ptx::float2_to_bf16x2(v[0], v[1]), ptx::float2_to_bf16x2(v[2], v[3]),
                                      ptx::float2_to_bf16x2(v[4], v[5]), ptx::float2_to_bf16x2(v[6], v[7]));
            *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.y) + int64_t(m0 + row) * a.n + n0 + c) = packed;
        }
        tc::cluster_sync();                   // nobody leaves while others read its shared memory
    }

    tc::fence_before_thread_sync();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_thread_sync();
        tc::tmem_dealloc(tmem, 2 * BN);
    }
    if (threadIdx.x == 0) report(error_flag != 0, a.rows.status);
}

// ---------------------------------------------------------------------------------------- weight gradients
// A cluster owns (adapter, 256 columns of X); its CTAs take the adapter's row tiles in turn and add their sums through
// distributed shared memory in rank order. X is the A operand (its columns are the M of the product), t the B operand, written
// into shared memory by the epilogue warps as hi and lo. Row tiles in which the adapter does not occur are never read.
constexpr int kLoraWgradColumns = 256;
constexpr int kLoraMaxTileWords = 2048;       // bitmap of row tiles: 2048 * 32 tiles of 128 rows

__global__ void __launch_bounds__(192, 1)
lora_wgrad_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LoraWgradArgs a) {
    using namespace lora_detail;
    extern __shared__ uint8_t smem_raw[];
    constexpr int kMaxStages = 4, kM = kLoraWgradColumns;
    constexpr uint32_t kXBytes = kM * kLoraBlockK * 2;          // 64 tokens x 256 columns, blocks of 64 columns
    __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], ext_bar[kMaxStages], done_bar;
    __shared__ uint32_t tmem_slot, tile_bits[kLoraMaxTileWords];
    __shared__ volatile int error_flag;

    const int warp = threadIdx.x / 32, lane = ptx::lane_id();
    const int cluster = a.cluster, rank = blockIdx.x % cluster, item = blockIdx.x / cluster;
    const int m_tile = item % a.m_tiles, e = item / a.m_tiles, m0 = m_tile * kM;
    const int rp = math::align(a.rows.rank, 64), stages = a.num_stages;       // t's columns come in blocks of 64
    const uint32_t t_bytes = rp * 128u;       // hi; lo follows
    const int words = math::ceil_div(a.row_tiles, 32);
    uint8_t* smem = align_1024(smem_raw);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) ptx::mbarrier_init(&full_bar[s], 1), ptx::mbarrier_init(&empty_bar[s], 1), ptx::mbarrier_init(&ext_bar[s], 4);
        ptx::mbarrier_init(&done_bar, 1);
        ptx::fence_mbarrier_init();
        error_flag = 0;
        tc::prefetch_tensormap(&map_x);
    }
    for (int w = warp; w < words; w += 6) {
        const int tile = w * 32 + lane;
        const unsigned bits = __ballot_sync(0xffffffffu, tile < a.row_tiles and a.presence[int64_t(tile) * a.rows.num_adapters + e] != 0);
        if (lane == 0) tile_bits[w] = bits;
    }
    uint32_t columns = 32;
    while (columns < uint32_t(2 * rp)) columns *= 2;
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
        if (lane == 0) {
            walk([&](int token) {
                const int s = count % stages;
                if (error_flag or not ptx::mbarrier_wait(&empty_bar[s], ((count / stages) & 1) ^ 1)) { error_flag = 1; return false; }
                ptx::mbarrier_arrive_expect_tx(&full_bar[s], kXBytes);
                uint8_t* stage = smem + size_t(s) * a.stage_bytes;
                for (int i = 0; i < kM / 64; ++i) tc::tma_load_2d(stage + i * 8192, &map_x, m0 + 64 * i, token, &full_bar[s]);
                ++count;
                return true;
            });
            for (int i = max(0, count - stages); i < count; ++i) ptx::mbarrier_wait(&full_bar[i % stages], (i / stages) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = tc::make_idesc(tc::kFormatBF16, 128, rp, true, true);
            const uint64_t desc_x = tc::make_smem_desc(smem, 8192, 1024), desc_t = tc::make_smem_desc(smem + kXBytes, 8192, 1024);
            walk([&](int) {
                const int s = count % stages, phase = (count / stages) & 1;
                if (error_flag or not ptx::mbarrier_wait(&full_bar[s], phase) or not ptx::mbarrier_wait(&ext_bar[s], phase)) { error_flag = 1; return false; }
                tc::fence_after_thread_sync();
                const uint64_t step = uint64_t(s) * (a.stage_bytes >> 4);
                #pragma unroll
                for (int k = 0; k < kLoraBlockK / 16; ++k) {
                    #pragma unroll
                    for (int m = 0; m < 2; ++m) {               // 128 columns of X each, 16 KB apart
                        tc::mma_f16(tmem + m * rp, desc_x + step + m * 1024 + k * 128, desc_t + step + k * 128, idesc, count > 0 or k > 0);
                        tc::mma_f16(tmem + m * rp, desc_x + step + m * 1024 + k * 128, desc_t + step + (t_bytes >> 4) + k * 128, idesc, true);
                    }
                }
                tc::commit(&empty_bar[s]);
                ++count;
                return true;
            });
            tc::commit(&done_bar);
        }
    } else {
        // ------------------------------------------------------------------ writers of the B operand, then the epilogue
        const int id = threadIdx.x - 64, line = id & 63, side = id >> 6;
        bool ok = true;
        walk([&](int token) {
            const int s = count % stages, phase = (count / stages) & 1, row = token + line;
            const bool mine = adapter_of(a.rows, row) == e;
            uint8_t* stage = smem + size_t(s) * a.stage_bytes;
            ok = __all_sync(0xffffffffu, ptx::mbarrier_wait(&empty_bar[s], phase ^ 1));
            if (not ok) { error_flag = 1; return false; }
            for (int u = side; u < rp / 8; u += 2) {            // units of eight rank columns, shared by two threads
                float v[8];
                const bool there = mine and 8 * u < a.rows.rank;
                if (there) load8(a.t + int64_t(row) * a.rows.rank + 8 * u, v);
                #pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = there ? v[j] : 0.0f;
                uint4 hi, lo;
                split8(v, hi, lo);
                uint8_t* at = stage + kXBytes + (u / 8) * 8192 + line * 128 + (((u % 8) ^ (line & 7)) << 4);
                *reinterpret_cast<uint4*>(at) = hi;
                *reinterpret_cast<uint4*>(at + t_bytes) = lo;
            }
            // rows of other requests in this block: zeros instead of whatever they hold (0 * inf would be NaN)
            ok = ok and ptx::mbarrier_wait(&full_bar[s], phase);
            if (not mine and row < a.rows.num_rows)
                for (int i = side; i < kM / 64; i += 2)
                    for (int u = 0; u < 8; ++u) *reinterpret_cast<uint4*>(stage + i * 8192 + line * 128 + u * 16) = make_uint4(0, 0, 0, 0);
            ptx::fence_proxy_async_smem();
            ok = __all_sync(0xffffffffu, ok);
            if (not ok) { error_flag = 1; return false; }
            if (lane == 0) ptx::mbarrier_arrive(&ext_bar[s]);
            ++count;
            return not __any_sync(0xffffffffu, error_flag != 0);
        });
        if (not ptx::mbarrier_wait(&done_bar, 0)) error_flag = 1;
        tc::fence_after_thread_sync();
        const int quarter = warp & 3;
        float* part = reinterpret_cast<float*>(smem);
        for (int m = 0; m < 2; ++m) {
            float* out = part + (m * 128 + quarter * 32 + lane) * (rp + 1);
            for (int c = 0; c < a.rows.rank; c += 16) {
                uint32_t r[16];
                tc::tmem_ld_32x16(tmem + (uint32_t(quarter * 32) << 16) + m * rp + c, r);
                tc::wait_ld();
                #pragma unroll
                for (int i = 0; i < 16; ++i) out[c + i] = count > 0 ? __uint_as_float(r[i]) : 0.0f;
            }
        }
        tc::fence_before_thread_sync();
    }
    __syncthreads();
    if (cluster > 1) tc::cluster_sync();
    bool any = false;
    for (int w = 0; w < words; ++w) any = any or tile_bits[w] != 0;
    if (any or not a.accumulate) {
        const float* part = reinterpret_cast<const float*>(smem);
        const int share = kM / cluster, first = rank * share, r_count = a.rows.rank;
        for (int i = threadIdx.x; i < share * r_count; i += 192) {
            // neighbouring threads write neighbouring addresses in either layout
            const int m = first + (a.rank_major ? i % share : i / r_count), r = a.rank_major ? i / share : i % r_count;
            if (m0 + m >= a.m) continue;
            float sum = 0.0f;
            if (cluster > 1) for (int q = 0; q < cluster; ++q) sum += ld_cluster(tc::map_to_cta(part + m * (rp + 1) + r, q));
            else sum = part[m * (rp + 1) + r];
            const int64_t at = a.rank_major ? (int64_t(e) * r_count + r) * a.m + m0 + m : (int64_t(e) * a.m + m0 + m) * r_count + r;
            if (a.out_fp32) {
                float* d = reinterpret_cast<float*>(a.d) + at;
                *d = a.accumulate ? *d + sum : sum;
            } else {
                reinterpret_cast<__nv_bfloat16*>(a.d)[at] = __float2bfloat16_rn(sum);
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
