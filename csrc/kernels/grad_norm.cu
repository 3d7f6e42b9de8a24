// Launchers of the gradient-norm kernels: the tensor list is cut into tables that fit a kernel's parameters.
#include <algorithm>
#include <vector>

#include <deep_ep/common/exception.hpp>
#include <deep_ep/kernels/grad_norm.cuh>

#include "api.hpp"
#include "early_launch.hpp"

namespace deep_ep::launch {

using namespace kernels;

namespace {

constexpr int kFewTensors = 64, kSomeTensors = 256;

// The shortest table that holds `count` tensors: a launch copies all of it
template <typename Launch>
auto with_table(int count, Launch launch) {
    if (count <= kFewTensors) return launch.template operator()<kFewTensors>();
    if (count <= kSomeTensors) return launch.template operator()<kSomeTensors>();
    return launch.template operator()<kGradMaxTensors>();
}

template <int kTensors>
int fill_table(GradTable<kTensors>& table, const GradTensor* tensors, int count) {
    int chunks = 0;
    for (int i = 0; i < count; ++i) {
        table.in[i] = tensors[i].in, table.out[i] = tensors[i].out, table.numel[i] = tensors[i].numel;
        table.in_type[i] = static_cast<uint8_t>(tensors[i].in_type), table.out_type[i] = static_cast<uint8_t>(tensors[i].out_type);
        table.first_chunk[i] = chunks;
        chunks += static_cast<int>(math::ceil_div<int64_t>(tensors[i].numel, kGradChunk));
    }
    table.first_chunk[count] = chunks, table.num_tensors = count;
    return chunks;
}

template <int kTensors>
int square_sum(const GradTensor* tensors, int count, double* partial, cudaStream_t stream) {
    GradTable<kTensors> table;
    const int grid = std::min(fill_table(table, tensors, count), kGradCtas);
    launch_kernel_as({grid, kGradThreads}, grad_square_sum_kernel<kTensors>, stream, table, GradNormArgs{partial});
    return grid;
}

template <int kTensors>
void clip(const GradTensor* tensors, int count, const GradClipArgs& args, cudaStream_t stream) {
    GradTable<kTensors> table;
    const int grid = std::min(fill_table(table, tensors, count), kGradCtas);
    launch_kernel_as({grid, kGradThreads}, grad_clip_kernel<kTensors>, stream, table, args);
}

}  // namespace

int grad_norm_max_sums(int num_tensors) { return math::ceil_div(num_tensors, kGradMaxTensors) * kGradCtas; }

int grad_square_sums(const std::vector<GradTensor>& tensors, double* partial, cudaStream_t stream) {
    int sums = 0;
    for (size_t i = 0; i < tensors.size(); i += kGradMaxTensors) {
        const int count = static_cast<int>(std::min<size_t>(kGradMaxTensors, tensors.size() - i));
        sums += with_table(count, [&]<int kTensors>() { return square_sum<kTensors>(tensors.data() + i, count, partial + sums, stream); });
    }
    return sums;
}

void grad_norm_finish(const GradClipArgs& args, cudaStream_t stream) { launch_kernel_as({1, kGradThreads}, grad_norm_finish_kernel, stream, args); }

void grad_clip(const std::vector<GradTensor>& tensors, GradClipArgs args, cudaStream_t stream) {
    for (size_t i = 0; i < tensors.size(); i += kGradMaxTensors) {
        const int count = static_cast<int>(std::min<size_t>(kGradMaxTensors, tensors.size() - i));
        with_table(count, [&]<int kTensors>() { clip<kTensors>(tensors.data() + i, count, args, stream); });
        args.norm = nullptr;
    }
}

}  // namespace deep_ep::launch
