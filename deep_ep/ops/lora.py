"""Low-rank adapters of many requests beside one shared projection, on tcgen05 kernels.

`lora_linear` is `dense_linear` with an adapter per row: `y[i] = x[i] W^T + scaling[e] (x[i] A_e^T) B_e^T`, `e` the row's
adapter. One call serves a batch whose rows belong to different requests (decode: every row another adapter; prefill: runs of
rows), in whatever order they come, and trains several adapters of one base model at once. The low-rank term is accumulated
into the shared product's own accumulator, so the result is rounded once. Nothing depends on the host knowing which adapters
occur: a call can be captured in a CUDA graph and replayed with other indices.

CPU tensors take the same formulas in plain torch.
"""
from typing import Optional, Union

import torch

from .._C_loader import _C

__all__ = ['lora_linear']


def _reference(x, w, lora_a, lora_b, idx, scaling):
    """Plain form in fp32 (CPU): rows are picked by adapter, so one adapter's values never meet another's rows."""
    dtype = x.dtype
    x, w, lora_a, lora_b = x.float(), w.float(), lora_a.float(), lora_b.float()      # once: their gradients are summed in fp32 too
    y = x @ w.t()
    for e in range(lora_a.size(0)):
        rows = torch.nonzero(idx == e).flatten()          # (an adapter without rows gets a gradient of zeros, as on the GPU)
        y = y.index_add(0, rows, scaling[e] * ((x[rows] @ lora_a[e].t()) @ lora_b[e].t()))
    return y.to(dtype)


def _weight_grad(x, t, idx, presence, parameter, rank_major):
    """Gradient of A (`rank_major`) or B; added to the parameter's fp32 `main_grad` where it has one."""
    main_grad = getattr(parameter, 'main_grad', None)
    out = torch.empty_like(parameter, memory_format=torch.contiguous_format) if main_grad is None else main_grad
    _C.lora_wgrad(x, t, idx, presence, out, rank_major, main_grad is not None)
    return out if main_grad is None else None


class _LoraLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, lora_a, lora_b, idx, scaling):
        y, t = _C.lora_forward(x, w, lora_a, lora_b, idx, scaling)
        ctx.save_for_backward(x, w, lora_a, lora_b, idx, scaling, t)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, lora_a, lora_b, idx, scaling, t = ctx.saved_tensors
        dy = dy.to(torch.bfloat16).contiguous()
        dx = dw = da = db = None
        want_x, want_w, want_a, want_b = ctx.needs_input_grad[:4]
        if want_x or want_a or want_b:
            dt, presence, dx = _C.lora_backward(dy, w, lora_a, lora_b, idx, scaling, want_x)
        if want_a:
            da = _weight_grad(x, dt, idx, presence, lora_a, True)
        if want_b:
            db = _weight_grad(dy, t, idx, presence, lora_b, False)
        if want_w:
            from .grouped_gemm import grouped_gemm_wgrad
            one = torch.full((1,), x.size(0), dtype=torch.int32, device=x.device)       # one group, all rows
            dw = torch.empty((1, *w.shape), dtype=w.dtype, device=w.device)
            grouped_gemm_wgrad(dy, x.contiguous(), dw, one, one, accumulate=False)
            dw = dw[0]
        return dx, dw, da, db, None, None


def lora_linear(x: torch.Tensor, w: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter_idx: torch.Tensor,
                scaling: Optional[Union[float, torch.Tensor]] = 1.0) -> torch.Tensor:
    """`x @ w.T + scaling[e] * (x @ lora_a[e].T) @ lora_b[e].T` per row, bf16 `[rows, N]`.

    `x [rows, K]`, `w [N, K]`, `lora_a [adapters, rank, K]`, `lora_b [adapters, N, rank]`, all bf16; `adapter_idx [rows]`
    int32 or int64, an index outside `[0, adapters)` (negative = none) leaves the row with the shared product; `scaling` one
    number or fp32 `[adapters]`. On a GPU K and N are multiples of 8 and the rank is a multiple of 8 up to 128 (pad smaller
    ranks with zero rows). Both products accumulate in fp32; the intermediate `x A^T` keeps 16 bits; `y` is rounded once.

    Gradients reach `x`, `lora_a` and `lora_b` (or their fp32 `main_grad`), and `w` if it wants one (K and N multiples of
    128 then). Infinities or NaN in a request's rows or adapter stay with the rows and adapter they belong to. The adapters'
    gradients read a row tile of 128 once per adapter that occurs in it, so long training batches are best ordered by adapter.
    A backward pass may be captured in a CUDA graph when no eager autograd graph of the same leaves is alive.
    """
    if not isinstance(scaling, torch.Tensor):
        scaling = torch.full((lora_a.size(0),), float(scaling), dtype=torch.float32, device=x.device)
    assert not scaling.requires_grad, 'scaling receives no gradient'
    if x.is_cuda:
        if adapter_idx.dim() == 1 and adapter_idx.size(0) > 1 and adapter_idx.stride(0) != 1:
            adapter_idx = adapter_idx.contiguous()
        if not (torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or lora_a.requires_grad or lora_b.requires_grad)):
            return _C.lora_forward(x, w, lora_a, lora_b, adapter_idx, scaling)[0]       # (which looks at every argument)
        if w.requires_grad:
            assert w.size(0) % 128 == 0 and w.size(1) % 128 == 0, 'the gradient of w needs K and N to be multiples of 128'
        return _LoraLinear.apply(x, w, lora_a, lora_b, adapter_idx, scaling)
    assert x.dim() == 2 and w.dim() == 2 and lora_a.dim() == 3 and lora_b.dim() == 3, 'x [rows, K], w [N, K], lora_a [E, rank, K], lora_b [E, N, rank]'
    rows, k = x.shape
    n, adapters, rank = w.size(0), lora_a.size(0), lora_a.size(1)
    assert w.size(1) == k and lora_a.size(2) == k and lora_b.shape == (adapters, n, rank), 'shapes of x, w, lora_a and lora_b do not agree'
    assert adapter_idx.shape == (rows,) and adapter_idx.dtype in (torch.int32, torch.int64), 'one int32 or int64 adapter index per row'
    assert all(t.dtype == torch.bfloat16 for t in (x, w, lora_a, lora_b)), 'operands are bf16'
    assert all(t.device == x.device for t in (w, lora_a, lora_b, adapter_idx, scaling)), 'all tensors of a call lie on one device'
    assert scaling.shape == (adapters,) and scaling.dtype == torch.float32, 'scaling is a number or fp32 [adapters]'
    return _reference(x, w, lora_a, lora_b, adapter_idx, scaling)
