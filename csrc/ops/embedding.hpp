// Torch-facing entry points of the embedding kernels: argument checks, outputs, workspaces.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <limits>
#include <optional>
#include <utility>

#include <deep_ep/common/exception.hpp>

#include "../kernels/api.hpp"
#include "autograd.hpp"

namespace deep_ep::ops {

inline kernels::EmbType embedding_type(const torch::Tensor& t) {
    switch (t.scalar_type()) {
        case torch::kBFloat16: return kernels::EmbType::kBF16;
        case torch::kFloat16: return kernels::EmbType::kFP16;
        case torch::kFloat32: return kernels::EmbType::kFP32;
        case torch::kFloat8_e4m3fn: return kernels::EmbType::kE4M3;
        default: EP_HOST_UNREACHABLE("embedding tables are bf16, fp16, fp32 or e4m3");
    }
}

// A matrix whose columns are contiguous; rows may lie further apart.
inline void check_rows(const torch::Tensor& t) {
    EP_HOST_ASSERT_MSG(t.is_cuda() and t.dim() == 2 and (t.size(1) <= 1 or t.stride(1) == 1) and t.stride(0) >= 0,
                       "a CUDA matrix with contiguous columns is needed");
    check_memory(t);
}

inline void check_ids(const torch::Tensor& idx, const torch::Tensor& with) {
    EP_HOST_ASSERT_MSG(idx.is_contiguous() and (idx.scalar_type() == torch::kInt64 or idx.scalar_type() == torch::kInt32),
                       "indices are contiguous int64 or int32");
    EP_HOST_ASSERT_MSG(idx.device() == with.device(), "all tensors of a call lie on one device");
    check_memory(idx);
}

constexpr int64_t kEmbMaxGradSize = std::numeric_limits<int>::max() / 2;         // rows, columns and tokens of a gradient

// [*idx.shape, hidden] = scaled rows of `table` (bf16 for an e4m3 table, else the table's type)
inline torch::Tensor lookup_rows(const torch::Tensor& table, const torch::Tensor& idx_in, double scale,
                                 const std::optional<torch::Tensor>& table_sf) {
    const auto idx = idx_in.contiguous();
    check_rows(table), check_ids(idx, table);
    const auto type = embedding_type(table);
    EP_HOST_ASSERT_MSG((type == kernels::EmbType::kE4M3) == table_sf.has_value(), "an e4m3 table comes with its scales, another without");
    EP_HOST_ASSERT(table.size(1) <= std::numeric_limits<int>::max());
    const c10::cuda::CUDAGuard guard(table.device());
    kernels::EmbLookupArgs a = {};
    a.table = table.data_ptr(), a.table_stride = table.stride(0);
    a.idx = idx.data_ptr(), a.idx64 = idx.scalar_type() == torch::kInt64;
    a.num_tokens = idx.numel(), a.num_rows = table.size(0), a.hidden = static_cast<int>(table.size(1));
    a.scale = static_cast<float>(scale);
    if (table_sf.has_value()) {
        check_rows(*table_sf);
        EP_HOST_ASSERT_MSG(a.hidden % 128 == 0 and table_sf->scalar_type() == torch::kFloat32 and table_sf->size(0) == a.num_rows and
                           table_sf->size(1) == a.hidden / 128 and table_sf->device() == table.device(),
                           "scales are fp32 [rows, hidden / 128], hidden a multiple of 128");
        a.table_sf = table_sf->data_ptr<float>(), a.sf_stride = table_sf->stride(0);
    }
    auto shape = idx.sizes().vec();
    shape.push_back(a.hidden);
    auto out = torch::empty(shape, table.options().dtype(
        type == kernels::EmbType::kE4M3 ? torch::kBFloat16 : table.scalar_type()));
    a.out = out.data_ptr();
    launch::embedding_lookup(a, type, c10::cuda::getCurrentCUDAStream());
    return out;
}

// out[v] (+)= scale * sum of dy[t] over idx[t] == v; `out` fp32 or of dy's type (a new one of dy's type without), `accumulate`
// only for fp32
inline torch::Tensor embedding_grad(const torch::Tensor& dy_in, const torch::Tensor& idx_in, int64_t rows, double scale,
                                    const std::optional<torch::Tensor>& out_in, bool accumulate) {
    EP_HOST_ASSERT_MSG(dy_in.is_cuda() and dy_in.dim() == 2 and rows >= 0 and (out_in.has_value() or not accumulate), "dy is a CUDA matrix; accumulation needs `out`");
    const auto dy = dy_in.size(1) > 1 and dy_in.stride(1) != 1 ? dy_in.contiguous() : dy_in;
    const auto idx = idx_in.contiguous();
    const auto out = out_in.has_value() ? *out_in : torch::empty({rows, dy.size(1)}, dy.options());
    check_rows(dy), check_rows(out), check_ids(idx, dy);
    refuse_tangent(dy_in), refuse_tangent(out);
    EP_HOST_ASSERT_MSG(out.size(0) == rows, "out is [num_rows, hidden]");
    EP_HOST_ASSERT_MSG(out.device() == dy.device(), "all tensors of a call lie on one device");
    EP_HOST_ASSERT_MSG(dy.size(0) == idx.numel() and dy.size(1) == out.size(1), "dy is [number of indices, hidden], out [rows, hidden]");
    EP_HOST_ASSERT_MSG(dy.scalar_type() == out.scalar_type() or out.scalar_type() == torch::kFloat32, "out is fp32 or of dy's type");
    EP_HOST_ASSERT_MSG(not accumulate or out.scalar_type() == torch::kFloat32, "only an fp32 gradient is accumulated into");
    EP_HOST_ASSERT_MSG(out.size(0) <= 1 or out.stride(0) >= out.size(1), "rows of out overlap");
    const auto range = [](const torch::Tensor& t) {
        const auto begin = reinterpret_cast<uintptr_t>(t.data_ptr());
        return std::pair(begin, begin + (t.numel() == 0 ? 0 : ((t.size(0) - 1) * t.stride(0) + t.size(1)) * t.element_size()));
    };
    const auto [dy_begin, dy_end] = range(dy);
    const auto [out_begin, out_end] = range(out);
    EP_HOST_ASSERT_MSG(out_end <= dy_begin or dy_end <= out_begin or out_begin == out_end or dy_begin == dy_end, "out shares memory with dy");
    EP_HOST_ASSERT_MSG(idx.numel() <= kEmbMaxGradSize and out.size(0) <= kEmbMaxGradSize and out.size(1) <= kEmbMaxGradSize,
                       "a gradient's rows, columns and tokens are below 2^30");
    const auto in_type = embedding_type(dy), out_type = embedding_type(out);
    EP_HOST_ASSERT(in_type != kernels::EmbType::kE4M3);
    const c10::cuda::CUDAGuard guard(dy.device());
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream();
    const int num_tokens = static_cast<int>(idx.numel()), num_rows = static_cast<int>(out.size(0)), hidden = static_cast<int>(out.size(1));
    if (num_rows == 0 or hidden == 0) return out;
    if (out_in.has_value()) mark_written(out);

    kernels::EmbGradArgs g = {};
    g.dy = dy.data_ptr(), g.dy_stride = dy.stride(0);
    g.num_tokens = num_tokens, g.num_rows = num_rows, g.hidden = hidden, g.scale = static_cast<float>(scale);
    g.out = out.data_ptr(), g.out_stride = out.stride(0), g.accumulate = accumulate;
    if (num_tokens == 0) {
        if (not accumulate) at::Tensor(out.detach()).zero_();
        return out;
    }
    g.chunk = launch::embedding_grad_chunk(num_tokens, hidden), g.num_chunks = (num_tokens + g.chunk - 1) / g.chunk;
    // scratch of this call, from the caching allocator: freed in stream order, private to a graph that is being captured
    const int64_t sort_ints = launch::embedding_sort_workspace_ints(num_tokens), bitmap_ints = accumulate ? 0 : (num_rows + 31) / 32;
    const auto ints = torch::empty({sort_ints + bitmap_ints + 1 + g.num_chunks}, idx.options().dtype(torch::kInt32));
    const auto partial = torch::empty({g.num_chunks > 1 ? 2ll * g.num_chunks * hidden : 0}, dy.options().dtype(torch::kFloat32));
    g.partial = partial.data_ptr<float>();
    kernels::EmbSortArgs s = {};
    s.idx = idx.data_ptr(), s.idx64 = idx.scalar_type() == torch::kInt64, s.num_tokens = num_tokens, s.num_rows = num_rows;
    // a sum is written over the whole row, so only rows without a token need zeros
    s.touched = accumulate ? nullptr : reinterpret_cast<uint32_t*>(ints.data_ptr<int>() + sort_ints);
    g.touched = s.touched;
    s.num_crossing = g.num_crossing = ints.data_ptr<int>() + sort_ints + bitmap_ints, g.crossing = g.num_crossing + 1;
    launch::embedding_sort(s, ints.data_ptr<int>(), &g.ids, &g.order, stream);
    launch::embedding_grad(g, in_type, out_type, stream);
    return out;
}

class EmbeddingLookup : public torch::autograd::Function<EmbeddingLookup> {
public:
    static torch::Tensor forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& table, const torch::Tensor& idx, double scale) {
        ctx->save_for_backward({idx});
        ctx->saved_data["table"] = table;        // the parameter itself, for its `main_grad`; its values may change before the backward pass
        ctx->saved_data["scale"] = scale;
        return lookup_rows(table, idx, scale, std::nullopt);
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
        const bool again = at::GradMode::is_enabled();           // the gradient is to be differentiated in turn: refused where that happens
        torch::autograd::variable_list out(3);
        {
            const at::NoGradGuard no_grad;
            const auto table = ctx->saved_data["table"].toTensor();
            const auto idx = ctx->get_saved_variables()[0].reshape({-1}), dy = grads[0].reshape({idx.numel(), table.size(1)});
            const double scale = ctx->saved_data["scale"].toDouble();
            const auto buffer = main_grad(table);
            const auto dtable = embedding_grad(dy, idx, table.size(0), scale, buffer, buffer.has_value());
            if (not buffer.has_value()) out[0] = dtable;
        }
        if (again) refuse_second_derivatives(out, "embedding_lookup is differentiable once");
        return out;
    }
};

inline torch::Tensor embedding_lookup(const torch::Tensor& table, const torch::Tensor& idx, double scale, const std::optional<torch::Tensor>& table_sf) {
    refuse_tangent(table);
    if (not at::GradMode::is_enabled() or not table.requires_grad() or table_sf.has_value()) return lookup_rows(table, idx, scale, table_sf);
    check_rows(table);
    EP_HOST_ASSERT_MSG(idx.numel() <= kEmbMaxGradSize and table.size(0) <= kEmbMaxGradSize and table.size(1) <= kEmbMaxGradSize,
                       "a gradient's rows, columns and tokens are below 2^30");
    return EmbeddingLookup::apply(table, idx, scale);
}

inline void register_embedding(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("embedding_lookup", &embedding_lookup, py::arg("table"), py::arg("idx"), py::arg("scale") = 1.0, py::arg("table_sf") = py::none());
    m.def("embedding_grad", &embedding_grad, py::arg("dy"), py::arg("idx"), py::arg("num_rows"), py::arg("scale") = 1.0,
          py::arg("out") = py::none(), py::arg("accumulate") = false);
}

}  // namespace deep_ep::ops
