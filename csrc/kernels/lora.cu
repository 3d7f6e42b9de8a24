// Launchers of the adapter kernels: tensor maps, cluster sizes and tiles by problem size.
#include <algorithm>

#include <deep_ep/common/exception.hpp>
#include <deep_ep/kernels/lora.cuh>

#include "api.hpp"
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

// `early`: may begin while the kernel before it in the stream still runs (it waits for that kernel's results itself).
template <typename... Params, typename... Args>
void launch_clusters(void (*kernel)(Params...), int64_t grid, int threads, int cluster, int64_t smem, bool early, cudaStream_t stream, const Args&... args) {
    EP_HOST_ASSERT_MSG(grid < (int64_t(1) << 31), "too many tiles for one launch");
    CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(grid)), config.blockDim = dim3(threads);
    config.dynamicSmemBytes = static_cast<size_t>(smem), config.stream = stream;
    cudaLaunchAttribute attr[2];
    int count = 0;
    if (cluster > 1) {
        attr[count].id = cudaLaunchAttributeClusterDimension;
        attr[count].val.clusterDim.x = cluster, attr[count].val.clusterDim.y = attr[count].val.clusterDim.z = 1;
        ++count;
    }
    if (early) {
        attr[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[count].val.programmaticStreamSerializationAllowed = 1;
        ++count;
    }
    config.attrs = attr, config.numAttrs = count;
    CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, args...));
}

constexpr int64_t kRingBytes = 192 * 1024;

}  // namespace

void lora_shrink(LoraShrinkArgs args, const void* x, const void* a, cudaStream_t stream) {
    ensure_context_once_per_thread();
    args.rows.status = failure_word_checked();
    const int rows = args.rows.num_rows, rank = args.rows.rank;
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
    args.stage_bytes = kLoraTileRows * kLoraBlockK * 2 + args.chunk * rp * 128;
    args.num_stages = static_cast<int>(std::min<int64_t>(8, kRingBytes / args.stage_bytes));
    const int64_t part = int64_t(kLoraTileRows) * (rp + 4) * 4;                          // overlays the ring
    const int64_t smem = std::max<int64_t>(int64_t(args.num_stages) * args.stage_bytes, part) + 1024;
    const CUtensorMap map_x = make_map_2d(x, rows, args.k, kLoraBlockK, kLoraTileRows);
    const CUtensorMap map_a = args.mn_major ? make_map_3d(a, args.rows.num_adapters, args.k, rank, 64, 64)
                                            : make_map_3d(a, args.rows.num_adapters, rank, args.k, kLoraBlockK, rp);
    launch_clusters(lora_shrink_kernel, tiles * args.num_chunks * args.cluster, 192, args.cluster, smem, false, stream, map_x, map_a, args);
}

namespace {

template <int BN>
void launch_gemm(LoraGemmArgs args, const void* x, const void* w, int sms, cudaStream_t stream) {
    constexpr int kStages = BN == 256 ? 4 : 6;
    args.m_tiles = math::ceil_div(args.rows.num_rows, kLoraTileRows), args.n_tiles = math::ceil_div(args.n, BN);
    const int64_t tiles = int64_t(args.m_tiles) * args.n_tiles;
    EP_HOST_ASSERT_MSG(tiles < (int64_t(1) << 30), "too many tiles for one launch");
    args.cluster = BN == 128 ? choose_cluster(tiles, math::ceil_div(args.k, kLoraBlockK), 4, sms) : 1;
    const int64_t grid = args.cluster > 1 ? tiles * args.cluster : std::min<int64_t>(tiles, sms);
    const int64_t smem = kStages * int64_t(kLoraTileRows + BN) * kLoraBlockK * 2 + 4 * 4096 + 1024;
    const auto& r = args.rows;
    const CUtensorMap map_x = make_map_2d(x, r.num_rows, args.k, kLoraBlockK, kLoraTileRows);
    const CUtensorMap map_w = args.mn_major ? make_map_2d(w, args.k, args.n, 64, kLoraBlockK) : make_map_2d(w, args.n, args.k, kLoraBlockK, 128);
    const CUtensorMap map_v = args.mn_major ? make_map_3d(args.v, r.num_adapters, r.rank, args.n, 64, 64)
                                            : make_map_3d(args.v, r.num_adapters, args.n, r.rank, 64, 128);
    const CUtensorMap map_y = make_map_out(args.y, r.num_rows, args.n, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2);
    launch_clusters(lora_gemm_kernel<BN>, grid, 320, args.cluster, smem, true, stream, map_x, map_w, map_v, map_y, args);
}

}  // namespace

void lora_gemm(LoraGemmArgs args, const void* x, const void* w, cudaStream_t stream) {
    ensure_context_once_per_thread();
    args.rows.status = failure_word_checked();
    const int sms = device_sms();
    const int64_t wide = int64_t(math::ceil_div(args.rows.num_rows, kLoraTileRows)) * math::ceil_div(args.n, 256);
    // 256 columns per tile as soon as that gives every SM a tile: half the shared-memory traffic per product
    if (wide >= sms) launch_gemm<256>(args, x, w, sms, stream);
    else launch_gemm<128>(args, x, w, sms, stream);
}

void lora_wgrad(LoraWgradArgs args, const void* x, cudaStream_t stream) {
    ensure_context_once_per_thread();
    args.rows.status = failure_word_checked();
    const int rp = math::align(args.rows.rank, 64);
    args.m_tiles = math::ceil_div(args.m, kLoraWgradColumns);
    args.row_tiles = math::ceil_div(args.rows.num_rows, kLoraTileRows);
    EP_HOST_ASSERT_MSG(args.row_tiles <= kLoraMaxTileWords * 32, "too many rows for one call");
    const int adapters = std::min(args.rows.num_adapters, args.rows.num_rows);           // that can have rows at all
    const int blocks = math::ceil_div(args.rows.num_rows, kLoraBlockK);
    args.cluster = choose_cluster(int64_t(args.m_tiles) * adapters, math::ceil_div(blocks, adapters), 2, device_sms());
    args.stage_bytes = kLoraWgradColumns * kLoraBlockK * 2 + 2 * rp * 128;
    args.num_stages = static_cast<int>(std::min<int64_t>(4, kRingBytes / args.stage_bytes));
    const int64_t part = int64_t(kLoraWgradColumns) * (rp + 1) * 4;                      // overlays the ring
    const int64_t smem = std::max<int64_t>(int64_t(args.num_stages) * args.stage_bytes, part) + 1024;
    const CUtensorMap map_x = make_map_2d(x, args.rows.num_rows, args.m, 64, kLoraBlockK);
    launch_clusters(lora_wgrad_kernel, int64_t(args.m_tiles) * args.rows.num_adapters * args.cluster, 192, args.cluster, smem, false, stream, map_x, args);
}

}  // namespace deep_ep::launch
