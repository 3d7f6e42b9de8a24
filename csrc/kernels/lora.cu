// Launchers of the adapter kernels: tensor maps, cluster sizes and tiles by problem size.
#include <algorithm>

#include <deep_ep/common/exception.hpp>
#include <deep_ep/kernels/lora.cuh>

#include "api.hpp"
#include "early_launch.hpp"
#include "gemm_host.hpp"

namespace deep_ep::launch {

using namespace kernels;

namespace {

int device_sms() {
    int device = 0, sms = 0;
    CUDA_CHECK(cudaGetDevice(&device));
    CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    return sms;
}

// Largest power of two of CTAs per unit of work that the SMs can run side by side, with at least `least` K blocks for each
// and none of them empty.
int choose_cluster(int64_t units, int blocks, int least, int sms) {
    int cluster = 1;
    while (cluster < kLoraMaxCluster and units * cluster * 2 <= sms and blocks >= cluster * 2 * least and
           (cluster * 2 - 1) * math::ceil_div(blocks, cluster * 2) < blocks)
        cluster *= 2;
    return cluster;
}

constexpr int64_t kRingBytes = 192 * 1024;
// Up to this many products of x A^T, the kernel without tensor cores is ahead: its time is that of reading rows * rank * k
// elements of A from L2, the other's starts at what setting up a tile costs. Measured (it | tensor cores, us): forward as a
// whole, K 7168, N 4096, 8 adapters: 16 rows of rank 16 17.4 | 24.0, 96 of rank 32 (2^24.4) 27.4 | 27.9, 64 of rank 64 (2^24.8)
// 30.2 | 28.7, 128 of rank 64 (2^25.8) 36.4 | 30.2. With the rank contiguous (backward) it reads A in pieces of eight bytes; alone,
// K 7168: 64 rows of rank 8 (2^21.8) 6.8 | 9.6, 4 of rank 128 (2^21.8) 10.3 | 10.3, 16 of rank 64 (2^22.8) 17.1 | 9.6.
constexpr int64_t kFewProducts = int64_t(3) << 23, kFewProductsRankContiguous = int64_t(1) << 22;

// One row tile: the low-rank term is computed beside the shared product's stream of W while it has few elements of t, more of
// them when each reads little of V. Measured with K 7168, N 4096 (beside the stream | tensor cores, us): 8 adapters of rank 16:
// 64 rows 21.4 | 24.0, 128 rows 24.8 | 26.0; 64 adapters of rank 16: 128 rows 28.4 | 33.3; 8 of rank 32: 32 rows 20.8 | 24.0, 64 rows
// 27.4 | 25.3; 64 of rank 32: 32 rows 24.7 | 27.2, 64 rows 36.3 | 31.0; 8 of rank 64: 16 rows 21.9 | 23.9, 32 rows 30.2 | 26.1.
bool few_terms(const LoraRows& r) {
    const int64_t terms = int64_t(r.num_rows) * r.rank;
    return r.num_rows <= kLoraTileRows and (terms <= 1024 or terms * r.rank <= 32768);
}

}  // namespace

void lora_shrink(LoraShrinkArgs args, const void* x, const void* a, cudaStream_t stream) {
    ensure_context_once_per_thread();
    args.rows.status = failure_word_checked();
    const int rows = args.rows.num_rows, rank = args.rows.rank;
    if (rows <= kLoraTileRows and int64_t(rows) * rank * args.k <= (args.mn_major ? kFewProductsRankContiguous : kFewProducts)) {
        // (an SM divides its memory between cache and shared memory by the kernels on it: with the default, the next kernel's
        // CTAs, which need all of the latter, could not join before these have left)
        CUDA_CHECK(cudaFuncSetAttribute(lora_shrink_rows_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        launch_kernel_as({rows * int64_t(rank / 4), 256}, lora_shrink_rows_kernel, stream, static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(a), args);
        return;
    }
    const int rp = math::align(rank, args.mn_major ? 64 : 16);
    const int64_t tiles = math::ceil_div(rows, kLoraTileRows), sms = device_sms();
    const int distinct = std::min({args.rows.num_adapters, rows, kLoraTileRows});        // at most, per tile
    const int blocks = math::ceil_div(args.k, kLoraBlockK);
    // at most 256 accumulator columns and 32 KB of adapter blocks per stage
    const int most = std::min({256 / rp, int(32 * 1024 / (rp * 128)), 16, distinct});
    // First the CTAs of a tile share its contraction; when few tiles hold many adapters, those are dealt out too.
    args.cluster = choose_cluster(tiles, blocks, 4, static_cast<int>(sms));
    args.chunk = static_cast<int>(std::clamp<int64_t>(math::ceil_div<int64_t>(int64_t(distinct) * tiles * args.cluster, sms), 1, most));
    args.num_chunks = math::ceil_div(distinct, args.chunk);
    args.ring_bytes = kRingBytes;             // the partial sums of a cluster overlay it: at most 128 x 132 floats
    const int64_t smem = kRingBytes + 1024;
    const CUtensorMap map_x = make_map_2d(x, rows, args.k, kLoraBlockK, kLoraTileRows);
    const CUtensorMap map_a = args.mn_major ? make_map_3d(a, args.rows.num_adapters, args.k, rank, 64, 64)
                                            : make_map_3d(a, args.rows.num_adapters, rank, args.k, kLoraBlockK, rp);
    launch_kernel_as({tiles * args.num_chunks * args.cluster, 192, smem, args.cluster}, lora_shrink_kernel, stream, map_x, map_a, args);
}

namespace {

struct GemmMaps {
    CUtensorMap x, w, v, y;
};

// Boxes of 64 (K) x 128 over x and over K-major W and V; 64 x 64 where the columns of Y are contiguous
GemmMaps gemm_maps(const LoraGemmArgs& a, const void* x, const void* w) {
    const auto& r = a.rows;
    return {make_map_2d(x, r.num_rows, a.k, kLoraBlockK, kLoraTileRows),
            a.mn_major ? make_map_2d(w, a.k, a.n, 64, kLoraBlockK) : make_map_2d(w, a.n, a.k, kLoraBlockK, 128),
            a.mn_major ? make_map_3d(a.v, r.num_adapters, r.rank, a.n, 64, 64) : make_map_3d(a.v, r.num_adapters, a.n, r.rank, 64, 128),
            make_map_out(a.y, r.num_rows, a.n, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2)};
}

void launch_gemm(LoraGemmArgs args, const void* x, const void* w, int sms, cudaStream_t stream) {
    args.m_tiles = math::ceil_div(args.rows.num_rows, kLoraTileRows), args.n_tiles = math::ceil_div(args.n, kLoraGemmColumns);
    const int64_t tiles = int64_t(args.m_tiles) * args.n_tiles;
    EP_HOST_ASSERT_MSG(tiles < (int64_t(1) << 30), "too many tiles for one launch");
    args.cluster = choose_cluster(tiles, math::ceil_div(args.k, kLoraBlockK), 4, sms);
    const int64_t grid = args.cluster > 1 ? tiles * args.cluster : std::min<int64_t>(tiles, sms);
    const auto maps = gemm_maps(args, x, w);
    launch_kernel_as({grid, kLoraGemmThreads, kLoraGemmSmemBytes, args.cluster}, lora_gemm_kernel, stream, maps.x, maps.w, maps.v, maps.y, args);
}

void launch_gemm_pair(LoraGemmArgs args, const void* x, const void* w, int sms, cudaStream_t stream) {
    args.m_tiles = math::ceil_div(args.rows.num_rows, 2 * kLoraTileRows), args.n_tiles = math::ceil_div(args.n, 256), args.cluster = 1;
    const int64_t tiles = int64_t(args.m_tiles) * args.n_tiles;
    EP_HOST_ASSERT_MSG(tiles < (int64_t(1) << 30), "too many tiles for one launch");
    const auto maps = gemm_maps(args, x, w);
    launch_kernel_as({2 * std::min<int64_t>(tiles, sms / 2), kLoraGemmThreads, kLoraPairSmemBytes, 2}, lora_gemm_pair_kernel, stream, maps.x, maps.w, maps.v, maps.y, args);
}

// Few rows: columns per tile and CTAs per cluster by an estimate of the time. W comes from memory at 6.5 TB/s however it is
// cut; a CTA takes in at most about 110 KB per us of W and of x, which every column tile reads again; and a cluster costs two
// barriers (about 1 us) and the parts that each CTA sends to the others, at about 15 KB per us. Measured with W [4096, 7168]:
// 64 columns by two CTAs took 15.1 / 15.4 / 17.1 us for 1 / 32 / 128 rows, 128 columns by four 14.8 / 17.1 / 18.5 us (32 columns and
// no cluster 17.6 to 25 us: too many small blocks per CTA). Stages of up to 48 KB: fewer, larger steps leave the issuing warps
// ahead of memory.
bool launch_gemm_few(const LoraGemmArgs& g, const void* x, const void* w, int sms, cudaStream_t stream) {
    LoraGemmFewArgs args = {};
    args.rows = g.rows, args.k = g.k, args.n = g.n, args.mn_major = g.mn_major, args.t = g.t, args.v = g.v, args.y = g.y;
    args.x_box_rows = math::align(g.rows.num_rows, 8);
    const int blocks = math::ceil_div(g.k, kLoraBlockK);
    double best = 0;
    for (int bn = 64; bn <= 128; bn *= 2) {
        const int64_t tiles = math::ceil_div(g.n, bn);
        if (tiles > sms) continue;
        const int block_bytes = (args.x_box_rows + bn) * kLoraBlockK * 2, sub = std::clamp(48 * 1024 / block_bytes, 1, 4);
        const int cluster = choose_cluster(tiles, math::ceil_div(blocks, sub), 2, sms);
        const double stream_us = std::max(double(g.n) * g.k * 2 / 6.5e6, double(block_bytes) * blocks / cluster / 110e3);
        const double tail_us = cluster > 1 ? 1.0 + double(args.x_box_rows) * bn * 4 * (cluster - 1) / cluster / 15e3 : 0.0;
        if (best == 0 or stream_us + tail_us < best) best = stream_us + tail_us, args.block_n = bn, args.cluster = cluster, args.stage_blocks = sub;
    }
    if (best == 0) return false;
    const int64_t tiles = math::ceil_div(g.n, args.block_n);
    const int64_t part_bytes = int64_t(kLoraTileRows) * args.block_n * 4, budget = 225 * 1024 - 1024 - part_bytes;
    const int64_t stage = int64_t(args.stage_blocks) * (args.x_box_rows + args.block_n) * kLoraBlockK * 2;
    args.num_stages = static_cast<int>(std::min<int64_t>(32, budget / stage));
    const CUtensorMap map_x = make_map_2d(x, g.rows.num_rows, g.k, kLoraBlockK, args.x_box_rows);
    const CUtensorMap map_w = g.mn_major ? make_map_2d(w, g.k, g.n, 64, kLoraBlockK) : make_map_2d(w, g.n, g.k, kLoraBlockK, args.block_n);
    launch_kernel_as({tiles * args.cluster, 320, args.num_stages * stage + part_bytes + 1024, args.cluster}, lora_gemm_few_kernel, stream, map_x, map_w, args);
    return true;
}

}  // namespace

void lora_gemm(LoraGemmArgs args, const void* x, const void* w, cudaStream_t stream) {
    ensure_context_once_per_thread();
    args.rows.status = failure_word_checked();
    const int sms = device_sms();
    if (few_terms(args.rows) and launch_gemm_few(args, x, w, sms, stream)) return;
    // A wave of 256 x 256 tiles by pairs of CTAs takes about 1.5 times as long as one of 128 x 128 tiles by single ones. Measured
    // with K 4096, N 4096, rank 16 (pairs | single, us): 512 rows 37.8 | 31.5, 768 38.0 | 41.0, 1280 60.5 | 64.4, 8192 209 | 300.
    const int64_t rows = args.rows.num_rows;
    const int64_t tiles = math::ceil_div<int64_t>(rows, kLoraTileRows) * math::ceil_div(args.n, kLoraGemmColumns);
    const int64_t pair_tiles = math::ceil_div<int64_t>(rows, 2 * kLoraTileRows) * math::ceil_div(args.n, 256);
    if (sms >= 2 and 3 * math::ceil_div<int64_t>(pair_tiles, sms / 2) <= 2 * math::ceil_div<int64_t>(tiles, sms)) launch_gemm_pair(args, x, w, sms, stream);
    else launch_gemm(args, x, w, sms, stream);
}

void lora_wgrad(LoraWgradArgs args, const void* x, cudaStream_t stream) {
    ensure_context_once_per_thread();
    args.rows.status = failure_word_checked();
    const int half = args.rows.rank <= 32 ? 32 : math::align(args.rows.rank, 64);         // columns of hi, as many of lo
    args.m_tiles = math::ceil_div(args.m, kLoraWgradColumns);
    args.row_tiles = math::ceil_div(args.rows.num_rows, kLoraTileRows);
    EP_HOST_ASSERT_MSG(args.row_tiles <= kLoraMaxTileWords * 32, "too many rows for one call");
    const int adapters = std::min(args.rows.num_adapters, args.rows.num_rows);           // that can have rows at all
    const int blocks = math::ceil_div(args.rows.num_rows, kLoraBlockK);
    args.cluster = choose_cluster(int64_t(args.m_tiles) * adapters, math::ceil_div(blocks, adapters), 2, device_sms());
    args.stage_bytes = kLoraWgradColumns * kLoraBlockK * 2 + 2 * half * 128;
    args.num_stages = static_cast<int>(std::min<int64_t>(4, kRingBytes / args.stage_bytes));
    const int64_t part = int64_t(kLoraWgradColumns) * (math::align(args.rows.rank, 16) + 4) * 4;                      // overlays the ring
    const int64_t smem = std::max<int64_t>(int64_t(args.num_stages) * args.stage_bytes, part) + 1024;
    const CUtensorMap map_x = make_map_2d(x, args.rows.num_rows, args.m, 64, kLoraBlockK);
    const LaunchShape shape = {int64_t(args.m_tiles) * args.rows.num_adapters * args.cluster, 320, smem, args.cluster, false};
    if (args.rows.rank <= 32) launch_kernel_as(shape, lora_wgrad_kernel<2>, stream, map_x, args);
    else if (args.rows.rank <= 64) launch_kernel_as(shape, lora_wgrad_kernel<4>, stream, map_x, args);
    else launch_kernel_as(shape, lora_wgrad_kernel<kLoraMaxRank / 16>, stream, map_x, args);
}

}  // namespace deep_ep::launch
