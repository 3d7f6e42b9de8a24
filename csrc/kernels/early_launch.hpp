// Kernel launches with clusters and programmatic dependent launch.
#pragma once

#include <cuda_runtime.h>

#include <deep_ep/common/exception.hpp>

namespace deep_ep::launch {

struct LaunchShape {
    int64_t grid;
    int threads;
    int64_t smem = 0;
    int cluster = 1;
    bool early = true;        // may be set up, and begin, while the kernel before it in the stream still runs
};

// `early` kernels wait themselves (`cudaGridDependencySynchronize`) before they touch anything that earlier work in the stream
// reads or writes. A kernel lets the next one begin (`cudaTriggerProgrammaticLaunchCompletion`) only after its own such wait: the next
// one may be any kernel, and its wait is for this one.
// One exception: the products of lora.cuh load x and W before they wait. That is sound only behind a kernel that writes neither and
// keeps this rule, or is not early at all: when the product begins, that kernel has waited, so whatever made x and W is done.
// lora_shrink and its form for a few rows are launched directly before them; torch may put a fill of y in between. They write nothing
// before the wait: every accumulator waits for the list of its tile's adapters, or for t, and the warps that bring those have waited.
template <typename... Params, typename... Args>
void launch_kernel_as(const LaunchShape& shape, void (*kernel)(Params...), cudaStream_t stream, const Args&... args) {
    EP_HOST_ASSERT_MSG(shape.grid > 0 and shape.grid < (int64_t(1) << 31), "too many tiles for one launch");
    if (shape.smem > 48 * 1024)
        CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shape.smem)));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(shape.grid)), config.blockDim = dim3(shape.threads);
    config.dynamicSmemBytes = static_cast<size_t>(shape.smem), config.stream = stream;
    cudaLaunchAttribute attr[2];
    int count = 0;
    if (shape.cluster > 1) {
        attr[count].id = cudaLaunchAttributeClusterDimension;
        attr[count].val.clusterDim.x = shape.cluster, attr[count].val.clusterDim.y = attr[count].val.clusterDim.z = 1;
        ++count;
    }
    if (shape.early) {
        attr[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[count].val.programmaticStreamSerializationAllowed = 1;
        ++count;
    }
    config.attrs = attr, config.numAttrs = count;
    CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, args...));
}

}  // namespace deep_ep::launch
