// Host-side helpers shared by the launchers of the tensor-core kernels: tensor maps, the failure word, the context.
#pragma once

#include <cuda_runtime.h>

#include <deep_ep/common/exception.hpp>

#include "../runtime/driver.hpp"

namespace deep_ep::launch {

// Lets this thread make memory-management calls while a stream is being captured (they touch no captured stream).
struct RelaxedCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode)); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// 2-D bf16 tensor map over a row-major [rows, cols] matrix with a {box_cols, box_rows} box.
inline CUtensorMap make_map_2d(const void* base, int64_t rows, int64_t cols, int box_cols, int box_rows) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * 2};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t elem_strides[2] = {1, 1};
    EP_HOST_ASSERT(reinterpret_cast<uintptr_t>(base) % 16 == 0 and (cols * 2) % 16 == 0);
    DRV_CHECK(driver::cuTensorMapEncodeTiled()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides,
                                               box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
    return map;
}

// Tensor map over a result matrix [rows, cols] whose box is 32 rows of 128 bytes (128-byte swizzle): the unit an epilogue
// warp hands to the TMA store / reduce-add
inline CUtensorMap make_map_out(const void* base, int64_t rows, int64_t cols, CUtensorMapDataType type, int element_bytes) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * element_bytes};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / element_bytes), 32};
    const cuuint32_t elem_strides[2] = {1, 1};
    EP_HOST_ASSERT(reinterpret_cast<uintptr_t>(base) % 16 == 0 and (cols * element_bytes) % 16 == 0);
    DRV_CHECK(driver::cuTensorMapEncodeTiled()(&map, type, 2, const_cast<void*>(base), dims, strides, box, elem_strides,
                                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
    return map;
}

// 3-D bf16 tensor map over contiguous [depth, rows, cols] with a {box_cols, box_rows, 1} box: what lies beyond a matrix's
// rows or columns reads as zeros instead of its neighbour's elements.
inline CUtensorMap make_map_3d(const void* base, int64_t depth, int64_t rows, int64_t cols, int box_cols, int box_rows) {
    CUtensorMap map;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(depth)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols) * 2, static_cast<cuuint64_t>(rows * cols) * 2};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows), 1};
    const cuuint32_t elem_strides[3] = {1, 1, 1};
    EP_HOST_ASSERT(reinterpret_cast<uintptr_t>(base) % 16 == 0 and (cols * 2) % 16 == 0);
    DRV_CHECK(driver::cuTensorMapEncodeTiled()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides,
                                               box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
    return map;
}

// One word of mapped pinned host memory that the GEMM kernels set when one of their bounded waits ran out. It is looked
// at before every launch, so a kernel that gave up (and left its output incomplete) is reported at the next call at the
// latest instead of passing silently.
struct FailureWord {
    int* host = nullptr;
    int* device = nullptr;
    FailureWord() {
        const RelaxedCapture relaxed;         // the first call may come while a stream is being captured
        CUDA_CHECK(cudaHostAlloc(reinterpret_cast<void**>(&host), sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable));
        *host = 0;
        CUDA_CHECK(cudaHostGetDevicePointer(reinterpret_cast<void**>(&device), host, 0));
    }
};

inline int* failure_word_checked() {
    static FailureWord word;
    if (*static_cast<volatile int*>(word.host) != 0) {
        *word.host = 0;
        throw EPException("GEMM kernel", __FILE__, __LINE__,
                          "an earlier GEMM kernel gave up waiting on one of its barriers; its output is incomplete");
    }
    return word.device;
}

// The tensor-map encoder is a driver entry point and wants a current context on the calling thread; autograd worker
// threads may not have touched the runtime yet. Done once per thread, so that later launches (for instance inside a
// CUDA-graph capture, where memory-management calls are not allowed) make no such call.
inline void ensure_context_once_per_thread() {
    static thread_local bool ready = false;
    if (ready) return;
    const RelaxedCapture relaxed;
    CUDA_CHECK(cudaFree(nullptr));
    ready = true;
}

}  // namespace deep_ep::launch
