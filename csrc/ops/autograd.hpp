// What the native autograd nodes share. They are native because a pass over a small batch is a handful of launches of a few
// microseconds each, to which a node in Python adds about forty.
#pragma once

#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <memory>
#include <optional>

#include <deep_ep/common/exception.hpp>

namespace deep_ep::ops {

// The fp32 buffer that a parameter's gradient is added to, if its Python object carries one
inline std::optional<torch::Tensor> main_grad(const torch::Tensor& parameter) {
    const pybind11::gil_scoped_acquire gil;
    const auto object = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(parameter));
    const pybind11::object buffer = pybind11::getattr(object, "main_grad", pybind11::none());
    if (buffer.is_none()) return std::nullopt;
    EP_HOST_ASSERT_MSG(THPVariable_Check(buffer.ptr()), "`main_grad` is a tensor");
    return THPVariable_Unpack(buffer.ptr());
}

// Gradients that were asked for with a graph of their own: an error where somebody differentiates them
inline void refuse_second_derivatives(torch::autograd::variable_list& grads, const char* message) {
    for (auto& g : grads) {
        if (not g.defined()) continue;
        auto leaf = g.detach();
        leaf.set_requires_grad(true);
        g = (*std::make_shared<torch::autograd::DelayedError>(message, 1))({leaf})[0];
    }
}

// Fake tensors and subclasses that wrap other tensors say that they lie on a GPU and have no memory there: a kernel would be given
// address zero
inline void check_memory(const void* data, int64_t numel) {
    EP_HOST_ASSERT_MSG(data != nullptr or numel == 0, "a tensor without memory of its own (fake, or a wrapper of others)");
}
inline void check_memory(const torch::Tensor& t) { check_memory(t.const_data_ptr(), t.numel()); }

// The kernels carry no tangents; a tensor that has one is refused rather than answered without its derivative
inline void refuse_tangent(const torch::Tensor& t) {
    EP_HOST_ASSERT_MSG(not t._fw_grad(0).defined(), "no forward-mode differentiation on the GPU");
}

// A kernel has written (or, for clipping within the limit, may write) the tensor: as after a torch operation in place, a graph that has
// saved it refuses to go back. (Inference tensors have no version.)
inline void mark_written(const torch::Tensor& t) {
    if (not t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace deep_ep::ops
