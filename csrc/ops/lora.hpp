// Torch-facing entry points of the adapter kernels: argument checks and outputs.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <limits>
#include <optional>
#include <tuple>

#include <deep_ep/common/exception.hpp>

#include "../kernels/api.hpp"
#include "autograd.hpp"

namespace deep_ep::ops {

// The tensor as the TMA reads it: contiguous, on a 16-byte boundary (a copy where a view is neither)
inline torch::Tensor operand(const torch::Tensor& t, int dims, const torch::Tensor& with, torch::ScalarType type = torch::kBFloat16) {
    EP_HOST_ASSERT_MSG(t.is_cuda() and t.dim() == dims and t.scalar_type() == type, "CUDA tensors of the documented types and shapes");
    EP_HOST_ASSERT_MSG(t.device() == with.device(), "all tensors of a call lie on one device");
    for (int i = 0; i < dims; ++i) EP_HOST_ASSERT_MSG(t.size(i) <= std::numeric_limits<int>::max() / 2, "sizes above 2^30");
    const auto c = t.contiguous();
    check_memory(c);
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

inline kernels::LoraRows adapter_rows(const torch::Tensor& idx, const torch::Tensor& with, int64_t num_adapters, int64_t rank) {
    EP_HOST_ASSERT_MSG(idx.dim() == 1 and (idx.size(0) <= 1 or idx.stride(0) == 1) and idx.device() == with.device() and
                       (idx.scalar_type() == torch::kInt32 or idx.scalar_type() == torch::kInt64), "adapter indices are int32 or int64 [rows]");
    EP_HOST_ASSERT_MSG(idx.size(0) == with.size(0), "one adapter index per row");
    EP_HOST_ASSERT_MSG(num_adapters >= 1 and rank >= 8 and rank % 8 == 0 and rank <= kernels::kLoraMaxRank, "ranks are multiples of 8 up to 128");
    return {idx.data_ptr(), idx.scalar_type() == torch::kInt64, static_cast<int>(idx.size(0)), static_cast<int>(num_adapters), static_cast<int>(rank), nullptr};
}

// t fp32 [rows, rank] = scaling[e] * x . A_e^T, and presence uint8 [row tiles, adapters] where it is wanted. `transposed`: A is
// [adapters, k, rank]. Operands as `operand` leaves them.
inline torch::Tensor lora_shrink(const torch::Tensor& x, const torch::Tensor& a, const torch::Tensor& idx, const torch::Tensor& scaling, bool transposed,
                                 const std::optional<torch::Tensor>& presence) {
    const int64_t k = x.size(1), rank = transposed ? a.size(2) : a.size(1);
    EP_HOST_ASSERT_MSG((transposed ? a.size(1) : a.size(2)) == k and k >= 8 and k % 8 == 0, "contraction lengths agree and are multiples of 8");
    EP_HOST_ASSERT_MSG(scaling.size(0) == a.size(0), "one scaling per adapter");
    kernels::LoraShrinkArgs args = {};
    args.rows = adapter_rows(idx, x, a.size(0), rank);
    args.k = static_cast<int>(k), args.mn_major = transposed, args.scaling = scaling.data_ptr<float>();
    auto t = torch::empty({x.size(0), rank}, x.options().dtype(torch::kFloat32));
    args.t = t.data_ptr<float>(), args.presence = presence.has_value() ? presence->data_ptr<uint8_t>() : nullptr;
    if (x.size(0) > 0) launch::lora_shrink(args, x.data_ptr(), a.data_ptr(), c10::cuda::getCurrentCUDAStream());
    return t;
}

// y = x . W^T + t . V_e^T; `transposed`: W is [k, n] and V [adapters, rank, n] (the data gradient), else [n, k] and [adapters, n, rank].
// Its kernel begins beside the one before it in the stream and loads x and W before it waits (see early_launch.hpp): that one has to
// be `lora_shrink`'s, with no launch that writes x or W (a copy of an operand, say) in between.
inline torch::Tensor lora_gemm_after_shrink(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& t, const torch::Tensor& v,
                                            const torch::Tensor& idx, bool transposed) {
    const int64_t k = x.size(1), n = transposed ? w.size(1) : w.size(0), rank = t.size(1);
    kernels::LoraGemmArgs args = {};
    args.rows = adapter_rows(idx, x, v.size(0), rank);
    args.k = static_cast<int>(k), args.n = static_cast<int>(n), args.mn_major = transposed;
    auto y = torch::empty({x.size(0), n}, x.options());
    args.t = t.data_ptr<float>(), args.v = v.data_ptr(), args.y = y.data_ptr();
    if (x.size(0) > 0) launch::lora_gemm(args, x.data_ptr(), w.data_ptr(), c10::cuda::getCurrentCUDAStream());
    return y;
}

inline void check_adapters(const torch::Tensor& w, const torch::Tensor& a, const torch::Tensor& b) {
    const int64_t n = w.size(0), k = w.size(1);
    EP_HOST_ASSERT_MSG(k >= 8 and k % 8 == 0 and n >= 8 and n % 8 == 0, "K and N are multiples of 8");
    EP_HOST_ASSERT_MSG(a.size(0) == b.size(0) and a.size(2) == k and b.size(1) == n and b.size(2) == a.size(1),
                       "w [N, K], a [adapters, rank, K], b [adapters, N, rank]");
}

// (y, t) of the forward pass
inline std::tuple<torch::Tensor, torch::Tensor> lora_forward(const torch::Tensor& x_in, const torch::Tensor& w_in, const torch::Tensor& a_in,
                                                             const torch::Tensor& b_in, const torch::Tensor& idx, const torch::Tensor& scaling_in) {
    const c10::cuda::OptionalCUDAGuard guard(x_in.is_cuda() ? std::optional(x_in.device()) : std::nullopt);
    const auto x = operand(x_in, 2, x_in), w = operand(w_in, 2, x_in), a = operand(a_in, 3, x_in), b = operand(b_in, 3, x_in);
    const auto scaling = operand(scaling_in, 1, x_in, torch::kFloat32);
    check_adapters(w, a, b);
    const auto t = lora_shrink(x, a, idx, scaling, false, std::nullopt);
    return {lora_gemm_after_shrink(x, w, t, b, idx, false), t};
}

// (dt, presence, dx or nothing) of the backward pass
inline std::tuple<torch::Tensor, torch::Tensor, std::optional<torch::Tensor>> lora_backward(
        const torch::Tensor& dy_in, const torch::Tensor& w_in, const torch::Tensor& a_in, const torch::Tensor& b_in, const torch::Tensor& idx,
        const torch::Tensor& scaling_in, bool want_dx) {
    const c10::cuda::OptionalCUDAGuard guard(dy_in.is_cuda() ? std::optional(dy_in.device()) : std::nullopt);
    const auto dy = operand(dy_in, 2, dy_in), w = operand(w_in, 2, dy_in), a = operand(a_in, 3, dy_in), b = operand(b_in, 3, dy_in);
    const auto scaling = operand(scaling_in, 1, dy_in, torch::kFloat32);
    check_adapters(w, a, b);
    auto presence = torch::empty({(dy.size(0) + kernels::kLoraTileRows - 1) / kernels::kLoraTileRows, b.size(0)}, dy.options().dtype(torch::kUInt8));
    const auto dt = lora_shrink(dy, b, idx, scaling, true, presence);
    std::optional<torch::Tensor> dx;
    if (want_dx) dx = lora_gemm_after_shrink(dy, w, dt, a, idx, true);
    return {dt, presence, dx};
}

// out[e] (+)= sum over the rows of adapter e of t[row]^T x[row]: [adapters, rank, m] (`rank_major`) or [adapters, m, rank]
inline void lora_wgrad(const torch::Tensor& x_in, const torch::Tensor& t_in, const torch::Tensor& idx, const torch::Tensor& presence,
                       const torch::Tensor& out, bool rank_major, bool accumulate) {
    const c10::cuda::OptionalCUDAGuard guard(x_in.is_cuda() ? std::optional(x_in.device()) : std::nullopt);
    const auto x = operand(x_in, 2, x_in), t = operand(t_in, 2, x_in, torch::kFloat32);
    EP_HOST_ASSERT_MSG(out.device() == x.device() and out.dim() == 3 and out.is_contiguous(), "a contiguous result on the operands' device");
    check_memory(out);
    EP_HOST_ASSERT_MSG(presence.device() == x.device() and presence.dim() == 2 and presence.is_contiguous() and presence.scalar_type() == torch::kUInt8, "presence of `lora_shrink`");
    const int64_t rank = t.size(1), m = x.size(1);
    EP_HOST_ASSERT_MSG(t.size(0) == x.size(0) and m >= 8 and m % 8 == 0, "one t per row, columns a multiple of 8");
    EP_HOST_ASSERT_MSG(out.size(1) == (rank_major ? rank : m) and out.size(2) == (rank_major ? m : rank), "the result's shape");
    EP_HOST_ASSERT_MSG(out.scalar_type() == torch::kFloat32 or (out.scalar_type() == torch::kBFloat16 and not accumulate), "fp32, or bf16 and overwritten");
    EP_HOST_ASSERT_MSG(out.scalar_type() == torch::kFloat32 or reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0, "a bf16 result starts on a 16-byte boundary");
    kernels::LoraWgradArgs args = {};
    args.rows = adapter_rows(idx, x, out.size(0), rank);
    EP_HOST_ASSERT(presence.size(1) == out.size(0) and presence.size(0) == (x.size(0) + kernels::kLoraTileRows - 1) / kernels::kLoraTileRows);
    if (x.size(0) == 0) {
        if (not accumulate) out.zero_();
        return;
    }
    mark_written(out);
    args.m = static_cast<int>(m), args.rank_major = rank_major;
    args.t = t.data_ptr<float>(), args.presence = presence.data_ptr<uint8_t>();
    args.d = out.data_ptr(), args.out_fp32 = out.scalar_type() == torch::kFloat32, args.accumulate = accumulate;
    launch::lora_wgrad(args, x.data_ptr(), c10::cuda::getCurrentCUDAStream());
}

// Gradient of a [N, K] weight: dy^T x, in the weight's type
inline torch::Tensor dense_weight_grad(const torch::Tensor& dy, const torch::Tensor& x, const torch::Tensor& w, bool pairs) {
    auto dw = torch::empty_like(w, w.options(), torch::MemoryFormat::Contiguous);
    if (x.size(0) == 0) return dw.zero_();
    const auto rows = torch::full({1}, x.size(0), x.options().dtype(torch::kInt32));          // one group, all rows
    kernels::GroupedGemmArgs args = {};
    args.mode = kernels::kModeWgrad, args.epilogue = kernels::kEpilogueStore, args.num_groups = 1, args.out_bf16 = true;
    args.psum = args.count = rows.data_ptr<int>();
    args.m = static_cast<int>(dy.size(1)), args.n = static_cast<int>(x.size(1)), args.d = dw.data_ptr();
    launch::grouped_gemm(args, dy.data_ptr(), dy.size(0), dy.size(1), x.data_ptr(), x.size(0), x.size(1), 0, c10::cuda::getCurrentCUDAStream(), pairs);
    return dw;
}

class LoraLinear : public torch::autograd::Function<LoraLinear> {
public:
    static torch::Tensor forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& a,
                                 const torch::Tensor& b, const torch::Tensor& idx, const torch::Tensor& scaling, bool pairs) {
        auto [y, t] = lora_forward(x, w, a, b, idx, scaling);
        ctx->save_for_backward({x, w, a, b, idx, scaling, t});
        // the parameters themselves, for their `main_grad`: what a hook on saved tensors (checkpointing) gives back is another tensor
        ctx->saved_data["a"] = a, ctx->saved_data["b"] = b;
        ctx->saved_data["pairs"] = pairs;
        return y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
        const bool again = at::GradMode::is_enabled();           // the gradients are to be differentiated in turn: refused where that happens
        torch::autograd::variable_list out(7);
        {
            const at::NoGradGuard no_grad;
            const auto saved = ctx->get_saved_variables();
            const auto &x = saved[0], &w = saved[1], &a = saved[2], &b = saved[3], &idx = saved[4], &scaling = saved[5], &t = saved[6];
            const c10::cuda::CUDAGuard guard(x.device());
            const auto dy = operand(grads[0].to(torch::kBFloat16), 2, x);
            const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_a = ctx->needs_input_grad(2), want_b = ctx->needs_input_grad(3);
            // gradient of A or B; added to the parameter's buffer where it has one
            const auto adapter_grad = [&](const torch::Tensor& rows, const torch::Tensor& low, const torch::Tensor& presence, const char* name, bool rank_major) {
                const auto parameter = ctx->saved_data[name].toTensor();
                const auto buffer = main_grad(parameter);
                const auto result = buffer.has_value() ? *buffer : torch::empty_like(parameter, parameter.options(), torch::MemoryFormat::Contiguous);
                lora_wgrad(rows, low, idx, presence, result, rank_major, buffer.has_value());
                return buffer.has_value() ? torch::Tensor() : result;
            };
            if (want_x or want_a or want_b) {
                const auto [dt, presence, dx] = lora_backward(dy, w, a, b, idx, scaling, want_x);
                if (want_x) out[0] = *dx;
                if (want_a) out[2] = adapter_grad(x, dt, presence, "a", true);
                if (want_b) out[3] = adapter_grad(dy, t, presence, "b", false);
            }
            if (want_w) out[1] = dense_weight_grad(dy, operand(x, 2, x), w, ctx->saved_data["pairs"].toBool());
        }
        if (again) refuse_second_derivatives(out, "lora_linear is differentiable once");
        return out;
    }
};

// y of the operator; `scalings` (fp32 [adapters]) goes before `scaling`
inline torch::Tensor lora_linear(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& idx_in,
                                 double scaling, const std::optional<torch::Tensor>& scalings, bool pairs) {
    EP_HOST_ASSERT_MSG(x.is_cuda() and a.dim() == 3 and idx_in.dim() == 1, "x is a CUDA matrix, a [adapters, rank, K], adapter indices [rows]");
    for (const auto* t : {&x, &w, &a, &b, &idx_in}) check_memory(*t);
    const c10::cuda::CUDAGuard guard(x.device());
    const auto idx = idx_in.contiguous();
    const auto s = scalings.has_value() ? *scalings : torch::full({a.size(0)}, scaling, x.options().dtype(torch::kFloat32).requires_grad(false));
    EP_HOST_ASSERT_MSG(not s.requires_grad(), "scaling receives no gradient");
    for (const auto* t : {&x, &w, &a, &b, &s}) refuse_tangent(*t);
    if (not at::GradMode::is_enabled() or not (x.requires_grad() or w.requires_grad() or a.requires_grad() or b.requires_grad()))
        return std::get<0>(lora_forward(x, w, a, b, idx, s));
    EP_HOST_ASSERT_MSG(not (a.requires_grad() or b.requires_grad()) or x.size(0) <= kernels::kLoraMaxGradRows, "gradients of a and b take up to 2^23 rows");
    EP_HOST_ASSERT_MSG(not w.requires_grad() or (w.dim() == 2 and w.size(0) % 128 == 0 and w.size(1) % 128 == 0), "the gradient of w needs K and N to be multiples of 128");
    return LoraLinear::apply(x, w, a, b, idx, s, pairs);
}

inline void register_lora(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("lora_linear", &lora_linear, py::arg("x"), py::arg("w"), py::arg("a"), py::arg("b"), py::arg("idx"), py::arg("scaling") = 1.0,
          py::arg("scalings") = py::none(), py::arg("gemm_pairs") = true);
}

}  // namespace deep_ep::ops
