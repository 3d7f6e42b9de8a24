// Torch-facing entry points of the gradient norm and clipping: argument checks, the tensor list, workspaces.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <vector>

#include <deep_ep/common/exception.hpp>

#include "../kernels/api.hpp"
#include "autograd.hpp"

namespace deep_ep::ops {

inline kernels::GradType gradient_type(const torch::Tensor& t) {
    switch (t.scalar_type()) {
        case torch::kBFloat16: return kernels::GradType::kBF16;
        case torch::kFloat16: return kernels::GradType::kFP16;
        case torch::kFloat32: return kernels::GradType::kFP32;
        default: EP_HOST_UNREACHABLE("gradients are bf16, fp16 or fp32");
    }
}

// The tensors of a Python list or tuple, without a copy of each: a step's list may hold hundreds of them
class TensorList {
    pybind11::object sequence;

public:
    explicit TensorList(const pybind11::object& object) {
        EP_HOST_ASSERT_MSG(PySequence_Check(object.ptr()), "a list or tuple of tensors");
        sequence = pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(object.ptr(), "a list or tuple of tensors"));
        for (size_t i = 0; i < size(); ++i) EP_HOST_ASSERT_MSG(THPVariable_Check(PySequence_Fast_GET_ITEM(sequence.ptr(), i)), "a list or tuple of tensors");
    }
    size_t size() const { return static_cast<size_t>(PySequence_Fast_GET_SIZE(sequence.ptr())); }
    const torch::Tensor& operator[](size_t i) const { return THPVariable_Unpack(PySequence_Fast_GET_ITEM(sequence.ptr(), i)); }
};

// The tensors as flat memory. Written tensors may share no memory with each other or, other than element for element, with
// a tensor that is read: two CTAs would then scale the same element.
inline std::vector<launch::GradTensor> gradient_list(const TensorList& grads, const TensorList* outs) {
    struct Range {
        uintptr_t begin, end;
        bool written;
    };
    std::vector<launch::GradTensor> list;
    std::vector<Range> ranges;
    list.reserve(grads.size());
    EP_HOST_ASSERT_MSG(grads.size() > 0, "an empty list has no device");
    EP_HOST_ASSERT_MSG(outs == nullptr or outs->size() == grads.size(), "one output per gradient");
    const auto device = grads[0].device();
    for (size_t i = 0; i < grads.size(); ++i) {
        const auto& g = grads[i];
        EP_HOST_ASSERT_MSG(g.is_cuda() and g.device() == device, "gradients lie on one CUDA device");
        EP_HOST_ASSERT_MSG(g.is_non_overlapping_and_dense(), "gradients are dense (no gaps, no element twice)");
        launch::GradTensor t = {g.const_data_ptr(), nullptr, g.numel(), gradient_type(g), gradient_type(g)};
        check_memory(t.in, t.numel);
        const auto begin = reinterpret_cast<uintptr_t>(t.in);
        if (outs != nullptr) {
            const auto& o = (*outs)[i];
            EP_HOST_ASSERT_MSG(o.device() == device and o.sizes() == g.sizes() and o.is_non_overlapping_and_dense() and
                               (o.strides() == g.strides() or g.numel() <= 1), "an output has its gradient's shape, strides and device");
            refuse_tangent(g), refuse_tangent(o);
            t.out = o.data_ptr(), t.out_type = gradient_type(o);
            check_memory(t.out, t.numel);
            const auto out_begin = reinterpret_cast<uintptr_t>(t.out);
            if (t.numel > 0) {
                ranges.push_back({out_begin, out_begin + o.nbytes(), true});
                if (t.in != t.out or t.in_type != t.out_type) ranges.push_back({begin, begin + g.nbytes(), false});
            }
        }
        if (t.numel > 0) list.push_back(t);
    }
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    uintptr_t end_any = 0, end_written = 0;
    for (const auto& r : ranges) {
        EP_HOST_ASSERT_MSG(r.begin >= (r.written ? end_any : end_written), "a written tensor shares memory with another tensor of the call");
        end_any = std::max(end_any, r.end);
        if (r.written) end_written = std::max(end_written, r.end);
    }
    return list;
}

// fp64 sums of squares whose total is the squared norm; at least one element
inline torch::Tensor square_sums(const std::vector<launch::GradTensor>& list, c10::Device device) {
    const c10::cuda::CUDAGuard guard(device);
    const auto options = torch::TensorOptions().dtype(torch::kFloat64).device(device);
    if (list.empty()) return torch::zeros({1}, options);
    auto sums = torch::empty({launch::grad_norm_max_sums(static_cast<int>(list.size()))}, options);
    const int count = launch::grad_square_sums(list, sums.data_ptr<double>(), c10::cuda::getCurrentCUDAStream());
    return sums.narrow(0, 0, count);
}

inline torch::Tensor grad_square_sums(const pybind11::object& grads) {
    const TensorList tensors(grads);
    const auto list = gradient_list(tensors, nullptr);
    return square_sums(list, tensors[0].device());
}

inline torch::Tensor grad_norm_finish(const torch::Tensor& sums) {
    EP_HOST_ASSERT(sums.is_cuda() and sums.is_contiguous() and sums.scalar_type() == torch::kFloat64);
    const c10::cuda::CUDAGuard guard(sums.device());
    auto norm = torch::empty({}, sums.options().dtype(torch::kFloat32));
    kernels::GradClipArgs args = {sums.data_ptr<double>(), static_cast<int>(sums.numel()), 0.0f, norm.data_ptr<float>(), 0};
    launch::grad_norm_finish(args, c10::cuda::getCurrentCUDAStream());
    return norm;
}

// the norm of one list
inline torch::Tensor grad_norm(const pybind11::object& grads) { return grad_norm_finish(grad_square_sums(grads)); }

// outs[i] = grads[i] * min(1, max_norm / (norm + 1e-6)), in place without `outs`; returns the norm
inline torch::Tensor grad_clip(const pybind11::object& grads, const pybind11::object& outs, const std::optional<torch::Tensor>& sums, double max_norm) {
    const TensorList tensors(grads);
    std::optional<TensorList> results;
    if (not outs.is_none()) results.emplace(outs);
    const auto list = gradient_list(tensors, results.has_value() ? &*results : &tensors);
    const auto device = tensors[0].device();
    const c10::cuda::CUDAGuard guard(device);
    const auto total = sums.has_value() ? *sums : square_sums(list, device);
    EP_HOST_ASSERT(total.device() == device and total.is_contiguous() and total.scalar_type() == torch::kFloat64);
    if (list.empty()) return grad_norm_finish(total);
    auto norm = torch::empty({}, total.options().dtype(torch::kFloat32));
    kernels::GradClipArgs args = {total.data_ptr<double>(), static_cast<int>(total.numel()), static_cast<float>(max_norm),
                                  norm.data_ptr<float>(), not results.has_value()};
    launch::grad_clip(list, args, c10::cuda::getCurrentCUDAStream());
    const TensorList& written = results.has_value() ? *results : tensors;
    for (size_t i = 0; i < written.size(); ++i) mark_written(written[i]);
    return norm;
}

inline void register_grad_norm(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("grad_square_sums", &grad_square_sums, py::arg("grads"));
    m.def("grad_norm_finish", &grad_norm_finish, py::arg("sums"));
    m.def("grad_norm", &grad_norm, py::arg("grads"));
    m.def("grad_clip", &grad_clip, py::arg("grads"), py::arg("outs"), py::arg("sums"), py::arg("max_norm"));
}

}  // namespace deep_ep::ops
