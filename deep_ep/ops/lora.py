"""Low-rank adapters of many requests beside one shared projection, on tcgen05 kernels.

`lora_linear` is `dense_linear` with an adapter per row: `y[i] = x[i] W^T + scaling[e] (x[i] A_e^T) B_e^T`, `e` the row's
adapter. One call serves a batch whose rows belong to different requests (decode: every row another adapter; prefill: runs of
rows), in whatever order they come, and trains several adapters of one base model at once. The low-rank term is accumulated
into the shared product's own accumulator, so the result is rounded once. Nothing depends on the host knowing which adapters
occur: a call can be captured in a CUDA graph and replayed with other indices.

CPU tensors take the same formulas in plain torch.
"""
from typing import Union

import torch

from .._C_loader import _C
from .grouped_gemm import MODE_WGRAD, _pairs

__all__ = ['lora_linear']


class _Widened(torch.autograd.Function):
    """`t.float()` of an adapter matrix. Its gradient is added to the matrix's `main_grad`, if it has one by then, as on the GPU."""
    generate_vmap_rule = True

    @staticmethod
    def forward(t):
        return t.float()

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.parameter, = inputs

    @staticmethod
    def backward(ctx, grad):
        main_grad = getattr(ctx.parameter, 'main_grad', None)
        if main_grad is None:
            return grad.to(ctx.parameter.dtype)
        with torch.no_grad():
            main_grad.add_(grad)

    @staticmethod
    def jvp(ctx, tangent):
        return tangent.float()


def _reference(x, w, lora_a, lora_b, idx, scaling):
    """Plain form in fp32 (CPU): rows are picked by adapter, so one adapter's values never meet another's rows."""
    dtype = x.dtype
    # once: their gradients are summed in fp32 too
    x, w, lora_a, lora_b = x.float(), w.float(), _Widened.apply(lora_a), _Widened.apply(lora_b)
    y = x @ w.t()
    for e in range(lora_a.size(0)):
        rows = torch.nonzero(idx == e).flatten()          # (an adapter without rows gets a gradient of zeros, as on the GPU)
        y = y.index_add(0, rows, scaling[e] * ((x[rows] @ lora_a[e].t()) @ lora_b[e].t()))
    return y.to(dtype)


def lora_linear(x: torch.Tensor, w: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter_idx: torch.Tensor,
                scaling: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """`x @ w.T + scaling[e] * (x @ lora_a[e].T) @ lora_b[e].T` per row, bf16 `[rows, N]`.

    `x [rows, K]`, `w [N, K]`, `lora_a [adapters, rank, K]`, `lora_b [adapters, N, rank]`, all bf16; `adapter_idx [rows]`
    int32 or int64, an index outside `[0, adapters)` (negative = none) leaves the row with the shared product; `scaling` one
    number or fp32 `[adapters]`. On a GPU K and N are multiples of 8 and the rank is a multiple of 8 up to 128 (pad smaller
    ranks with zero rows). Both products accumulate in fp32; the intermediate `x A^T` keeps 16 bits; `y` is rounded once.

    Gradients reach `x`, `lora_a` and `lora_b` (or their fp32 `main_grad`), and `w` if it wants one (K and N multiples of
    128 then). Infinities or NaN in a request's rows or adapter stay with the rows and adapter they belong to, whose
    results are infinite or NaN as the formulas say. The adapters' gradients read a row tile of 128 once per adapter that occurs
    in it, so long training batches are best ordered by adapter; they take up to 2^23 rows. A backward pass may be captured in a CUDA graph when no eager
    autograd graph of the same leaves is alive.
    """
    if x.is_cuda:
        # (the native call looks at every argument, and is the autograd node where a gradient is wanted)
        if isinstance(scaling, torch.Tensor):
            return _C.lora_linear(x, w, lora_a, lora_b, adapter_idx, 1.0, scaling, _pairs(MODE_WGRAD))
        return _C.lora_linear(x, w, lora_a, lora_b, adapter_idx, scaling, None, _pairs(MODE_WGRAD))
    if not isinstance(scaling, torch.Tensor):
        scaling = torch.full((lora_a.size(0),), float(scaling), dtype=torch.float32, device=x.device)
    assert not scaling.requires_grad, 'scaling receives no gradient'
    assert x.dim() == 2 and w.dim() == 2 and lora_a.dim() == 3 and lora_b.dim() == 3, 'x [rows, K], w [N, K], lora_a [E, rank, K], lora_b [E, N, rank]'
    rows, k = x.shape
    n, adapters, rank = w.size(0), lora_a.size(0), lora_a.size(1)
    assert w.size(1) == k and lora_a.size(2) == k and lora_b.shape == (adapters, n, rank), 'shapes of x, w, lora_a and lora_b do not agree'
    assert adapter_idx.shape == (rows,) and adapter_idx.dtype in (torch.int32, torch.int64), 'one int32 or int64 adapter index per row'
    assert all(t.dtype == torch.bfloat16 for t in (x, w, lora_a, lora_b)), 'operands are bf16'
    assert all(t.device == x.device for t in (w, lora_a, lora_b, adapter_idx, scaling)), 'all tensors of a call lie on one device'
    assert scaling.shape == (adapters,) and scaling.dtype == torch.float32, 'scaling is a number or fp32 [adapters]'
    return _reference(x, w, lora_a, lora_b, adapter_idx, scaling)
