// Launchers of the embedding kernels: vector widths by alignment, grids by size, the passes of the sort.
#include <algorithm>
#include <bit>

#include <deep_ep/common/exception.hpp>
#include <deep_ep/kernels/embedding.cuh>

#include "api.hpp"
#include "early_launch.hpp"

namespace deep_ep::launch {

using namespace kernels;

namespace {

bool aligned(const void* p, int64_t row_bytes, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 and row_bytes % bytes == 0; }

template <typename In, typename Out, int kElems, int kUnroll>
void launch_lookup(EmbLookupArgs a, cudaStream_t stream) {
    const int64_t slices = math::ceil_div(a.hidden / kElems, 32 * kUnroll);
    // item numbers are 32-bit in the kernel: very long inputs go in pieces
    const int64_t most = std::max<int64_t>(1, ((int64_t(1) << 31) - 8) / slices);
    for (int64_t done = 0, total = a.num_tokens; done < total; done += most) {
        EmbLookupArgs piece = a;
        piece.num_tokens = std::min(most, total - done);
        piece.idx = static_cast<const uint8_t*>(a.idx) + done * (a.idx64 ? 8 : 4);
        piece.out = static_cast<Out*>(a.out) + done * a.hidden;
        launch_kernel_as({(piece.num_tokens * slices + 7) / 8, 256}, embedding_lookup_kernel<In, Out, kElems, kUnroll>, stream, piece);
    }
}

// Widest access that both the table's rows and the result's allow: 16 bytes, 4 bytes, one element.
template <typename In, typename Out>
void choose_lookup(const EmbLookupArgs& a, cudaStream_t stream) {
    constexpr int kWide = 16 / sizeof(Out), kHalf = 4 / sizeof(Out);
    const auto fits = [&](int elems) {
        return a.hidden % elems == 0 and aligned(a.table, a.table_stride * sizeof(In), elems * int(sizeof(In))) and
               aligned(a.out, int64_t(a.hidden) * sizeof(Out), std::min(16, elems * int(sizeof(Out))));
    };
    if (fits(kWide)) {
        // few rows: one access per lane and item, so that a row is spread over more SMs. Measured with 7168 columns (one | four
        // accesses, us): 16 tokens 1.55 | 1.79, 128 1.80 | 1.80, 256 2.31 | 2.07, 8192 47.5 | 37.2.
        const bool small = a.num_tokens * math::ceil_div(a.hidden / kWide, 32) < 148 * 32;
        if (small) launch_lookup<In, Out, kWide, 1>(a, stream);
        else launch_lookup<In, Out, kWide, 4>(a, stream);
    } else if (kHalf > 1 and fits(kHalf)) {
        launch_lookup<In, Out, kHalf, 4>(a, stream);
    } else {
        launch_lookup<In, Out, 1, 4>(a, stream);
    }
}

}  // namespace

void embedding_lookup(const EmbLookupArgs& args, EmbType type, cudaStream_t stream) {
    if (args.num_tokens == 0 or args.hidden == 0) return;
    switch (type) {
        case EmbType::kBF16: return choose_lookup<__nv_bfloat16, __nv_bfloat16>(args, stream);
        case EmbType::kFP16: return choose_lookup<__half, __half>(args, stream);
        case EmbType::kFP32: return choose_lookup<float, float>(args, stream);
        case EmbType::kE4M3: return choose_lookup<__nv_fp8_e4m3, __nv_bfloat16>(args, stream);
    }
}

// ---------------------------------------------------------------------------------------- sort
namespace {

constexpr int kClusterKeys = 8 * kEmbClusterThreads * kEmbClusterMaxRounds;      // 65536 keys in one launch
constexpr int kKeysPerCta = 2048;

int sort_ctas(int num_tokens) { return std::min(148, math::ceil_div(num_tokens, kKeysPerCta)); }

// ids are 0 .. num_rows (num_rows = masked): as few passes of at most `most` bits as cover them, of equal width
void choose_digits(EmbSortArgs& a, int most) {
    const int bits = std::max(1, int(std::bit_width(static_cast<unsigned>(a.num_rows))));
    a.num_passes = math::ceil_div(bits, most);
    a.digit_bits = std::max(1, math::ceil_div(bits, a.num_passes));
}

template <int kRounds>
void sort_in_cluster(const EmbSortArgs& args, cudaStream_t stream) {
    constexpr int kKeys = kEmbClusterThreads * kRounds;
    const int bins = 1 << args.digit_bits;
    int cluster = 1;
    while (cluster * kKeys < args.num_tokens) cluster *= 2;
    const int smem = 4 * kKeys * 4 + 3 * bins * 4 + (kEmbClusterThreads / 32) * bins * 2;
    launch_kernel_as({cluster, kEmbClusterThreads, smem, cluster, args.touched == nullptr}, embedding_sort_cluster_kernel<kRounds>, stream, args);
}

}  // namespace

int64_t embedding_sort_workspace_ints(int num_tokens) {
    // two key and two value buffers, the counts of a pass
    return num_tokens <= kClusterKeys ? 2ll * num_tokens : 4ll * num_tokens + int64_t(sort_ctas(num_tokens)) * (1 << kEmbMaxDigitBits);
}

void embedding_sort(EmbSortArgs args, int* workspace, const int** ids, const int** order, cudaStream_t stream) {
    const int n = args.num_tokens;
    if (args.touched != nullptr) CUDA_CHECK(cudaMemsetAsync(args.touched, 0, (args.num_rows + 31ll) / 32 * 4, stream));
    if (n <= kEmbRankKeys) {
        args.keys[0] = workspace, args.vals[0] = workspace + n;
        // (after a memset there is no kernel to begin beside)
        launch_kernel_as({math::ceil_div(n, 32), kEmbRankThreads, math::align(n, 32) * 4, 1, args.touched == nullptr}, embedding_rank_kernel, stream, args);
        *ids = args.keys[0], *order = args.vals[0];
        return;
    }
    if (n <= kClusterKeys) {
        choose_digits(args, kEmbClusterDigitBits);
        args.keys[0] = workspace, args.vals[0] = workspace + n;
        // as few keys per thread as eight CTAs allow
        if (n <= 16 * kEmbClusterThreads) sort_in_cluster<2>(args, stream);
        else if (n <= 32 * kEmbClusterThreads) sort_in_cluster<4>(args, stream);
        else sort_in_cluster<8>(args, stream);
        *ids = args.keys[0], *order = args.vals[0];
        return;
    }
    choose_digits(args, kEmbMaxDigitBits);
    args.keys[0] = workspace, args.keys[1] = workspace + n;
    args.vals[0] = workspace + 2ll * n, args.vals[1] = workspace + 3ll * n;
    args.hist = workspace + 4ll * n;
    const int ctas = sort_ctas(n), warps = kEmbSortThreads / 32, bins = 1 << args.digit_bits;
    args.keys_per_warp = math::align(math::ceil_div(n, ctas * warps), 32);
    const int smem = (warps + 2) * bins * 4 + 128;
    for (args.pass = 0; args.pass < args.num_passes; ++args.pass) {
        embedding_sort_count_kernel<<<ctas, kEmbSortThreads, smem, stream>>>(args);
        embedding_sort_scatter_kernel<<<ctas, kEmbSortThreads, smem, stream>>>(args);
    }
    CUDA_CHECK(cudaGetLastError());
    *ids = args.keys[(args.num_passes - 1) & 1], *order = args.vals[(args.num_passes - 1) & 1];
}

// ---------------------------------------------------------------------------------------- gradient
int embedding_grad_chunk(int num_tokens, int hidden) {
    // Sorted positions per chunk: many make few runs that cross into the next chunk and have to be joined, few make enough items
    // for all SMs. Measured (8 | 16 | 32 | 64 positions, us): 16384 tokens with frequent repeats, 7168 columns 240 | 213 | 201 | 193;
    // 4096 without, 7168 columns 62 | 64 | 72 | 79; 5001 of 1003 columns 26 | 24 | 27 | 32; 500 of 7168 12.3 | 13.7 | 19.8 | 33.
    // Long inputs take more, so that a run over all of them is joined from at most 2048 pieces.
    int chunk = 64;
    const auto items = [&] { return int64_t(math::ceil_div(num_tokens, chunk)) * math::ceil_div(hidden, 128); };
    while ((chunk > 16 and items() < 148 * 64) or (chunk > 8 and items() < 148 * 16)) chunk /= 2;
    while (math::ceil_div(num_tokens, chunk) > 2048) chunk *= 2;
    return chunk;
}

namespace {

template <typename In, typename Out, int kElems, int kPacks, bool kAccumulate>
void launch_grad(const EmbGradArgs& a, cudaStream_t stream) {
    const int64_t slices = math::ceil_div(a.hidden, 32 * kElems * kPacks);
    const int64_t sums = int64_t(a.num_chunks) * slices, fills = a.accumulate ? 0 : a.num_rows;
    EP_HOST_ASSERT(sums < (int64_t(1) << 31));
    launch_kernel_as({(sums + fills + 7) / 8, 256}, embedding_grad_kernel<In, Out, kElems, kPacks, kAccumulate>, stream, a);
    if (a.num_chunks > 1) launch_kernel_as({148 * 6, 256}, embedding_grad_join_kernel<Out, kElems, kAccumulate>, stream, a);
}

template <typename In, typename Out>
void choose_grad(const EmbGradArgs& a, cudaStream_t stream) {
    constexpr int kWide = 16 / sizeof(In), kHalf = 4 / sizeof(In);
    const auto fits = [&](int elems) {
        return a.hidden % elems == 0 and aligned(a.dy, a.dy_stride * sizeof(In), elems * int(sizeof(In))) and
               aligned(a.out, a.out_stride * sizeof(Out), std::min(16, elems * int(sizeof(Out))));
    };
    const auto go = [&]<int kElems, int kPacks>() {
        if constexpr (sizeof(Out) == 4) {
            if (a.accumulate) return launch_grad<In, Out, kElems, kPacks, true>(a, stream);
        }
        launch_grad<In, Out, kElems, kPacks, false>(a, stream);
    };
    if (fits(kWide)) go.template operator()<kWide, 1>();
    else if (kHalf > 1 and fits(kHalf)) go.template operator()<kHalf, 2>();
    else go.template operator()<1, 4>();
}

}  // namespace

void embedding_grad(const EmbGradArgs& a, EmbType in, EmbType out, cudaStream_t stream) {
    if (a.hidden == 0) return;
    if (in == EmbType::kBF16 and out == EmbType::kBF16) return choose_grad<__nv_bfloat16, __nv_bfloat16>(a, stream);
    if (in == EmbType::kBF16 and out == EmbType::kFP32) return choose_grad<__nv_bfloat16, float>(a, stream);
    if (in == EmbType::kFP16 and out == EmbType::kFP16) return choose_grad<__half, __half>(a, stream);
    if (in == EmbType::kFP16 and out == EmbType::kFP32) return choose_grad<__half, float>(a, stream);
    if (in == EmbType::kFP32 and out == EmbType::kFP32) return choose_grad<float, float>(a, stream);
    EP_HOST_UNREACHABLE("gradient types");
}

}  // namespace deep_ep::launch
