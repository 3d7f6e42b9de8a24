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

namespace deep_ep::ops {

// The tensor as the TMA reads it: contiguous, on a 16-byte boundary (a copy where a view is neither)
inline torch::Tensor operand(const torch::Tensor& t, int dims, const torch::Tensor& with, torch::ScalarType type = torch::kBFloat16) {
    EP_HOST_ASSERT_MSG(t.is_cuda() and t.dim() == dims and t.scalar_type() == type, "CUDA tensors of the documented types and shapes");
    EP_HOST_ASSERT_MSG(t.device() == with.device(), "all tensors of a call lie on one device");
    for (int i = 0; i < dims; ++i) EP_HOST_ASSERT_MSG(t.size(i) <= std::numeric_limits<int>::max() / 2, "sizes above 2^30");
    const auto c = t.contiguous();
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
// Its kernel begins beside the one before it in the stream and waits for nothing but t: that one has to be `lora_shrink`'s,
// with no other launch (a copy of an operand, say) in between.
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
    args.m = static_cast<int>(m), args.rank_major = rank_major;
    args.t = t.data_ptr<float>(), args.presence = presence.data_ptr<uint8_t>();
    args.d = out.data_ptr(), args.out_fp32 = out.scalar_type() == torch::kFloat32, args.accumulate = accumulate;
    launch::lora_wgrad(args, x.data_ptr(), c10::cuda::getCurrentCUDAStream());
}

inline void register_lora(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("lora_forward", &lora_forward, py::arg("x"), py::arg("w"), py::arg("a"), py::arg("b"), py::arg("idx"), py::arg("scaling"));
    m.def("lora_backward", &lora_backward, py::arg("dy"), py::arg("w"), py::arg("a"), py::arg("b"), py::arg("idx"), py::arg("scaling"),
          py::arg("want_dx") = true);
    m.def("lora_wgrad", &lora_wgrad, py::arg("x"), py::arg("t"), py::arg("idx"), py::arg("presence"), py::arg("out"), py::arg("rank_major"),
          py::arg("accumulate") = false);
}

}  // namespace deep_ep::ops
