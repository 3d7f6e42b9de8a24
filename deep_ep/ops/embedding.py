"""Embedding lookup with scaling, and its gradient, on hand-written kernels.

Tables that live on one GPU, next to `EngramBuffer` (which gathers entries of tables sharded over ranks): the input
embedding of a model, or the local shard of an entry table during training. The index convention is Engram's: an index
outside the table (negative = masked) yields a row of zeros and receives no gradient, so a rank can hand in
`global_idx - rank * entries` and work on its own shard without masking first.

`embedding_lookup` is differentiable in the table. Its gradient is summed in fp32 over the tokens of an id in the order of
a stable sort, without atomics on values, so it has the same bits on every run. A table that carries an fp32
`main_grad` buffer has the gradient added there (as the grouped linear layers do with their weights) and autograd sees none.
CPU tensors take the same formulas in plain torch.
"""
from typing import Optional

import torch

from .._C_loader import _C

_TABLE_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _lookup(table: torch.Tensor, idx: torch.Tensor, scale: float, table_sf: Optional[torch.Tensor]) -> torch.Tensor:
    flat = idx.reshape(-1)
    valid = (flat >= 0) & (flat < table.size(0))
    rows = table.new_zeros((flat.numel(), table.size(1)), dtype=torch.float32)
    rows[valid] = table[flat[valid].long()].float()
    if table_sf is not None:
        rows[valid] = rows[valid] * table_sf[flat[valid].long()].repeat_interleave(128, dim=1)
    out = (rows * scale).to(torch.bfloat16 if table_sf is not None else table.dtype)
    return out.view(*idx.shape, table.size(1))


class _Lookup(torch.autograd.Function):          # CPU; the native call has its own
    @staticmethod
    def forward(ctx, table, idx, scale):
        ctx.save_for_backward(idx)
        ctx.table, ctx.scale = table, scale          # the parameter itself: its `main_grad` is looked up in the backward pass
        return _lookup(table, idx, scale, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        idx, = ctx.saved_tensors
        table = ctx.table
        dy = dy.reshape(idx.numel(), table.size(1))
        main_grad = getattr(table, 'main_grad', None)
        if main_grad is not None:
            embedding_grad(dy, idx, table.size(0), ctx.scale, out=main_grad, accumulate=True)
            return None, None, None
        return embedding_grad(dy, idx, table.size(0), ctx.scale), None, None


def embedding_lookup(table: torch.Tensor, idx: torch.Tensor, scale: float = 1.0,
                     table_sf: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`out[..., :] = table[idx[...]] * scale`, shape `[*idx.shape, hidden]`; indices outside `[0, rows)` give zeros.

    `table` is `[rows, hidden]` with contiguous columns (rows may lie further apart): bf16, fp16 or fp32, and the result has
    its type; or e4m3 with `table_sf`, fp32 `[rows, hidden / 128]` (the 1x128 scales of an FP8 entry table), and the result
    is bf16. `idx` is int64 or int32 of any shape. Products are taken in fp32 and rounded once. The gradient reaches `table`
    (not an e4m3 one) in its own type, or its fp32 `main_grad`, for fewer than 2^30 rows, columns and tokens; a backward pass may
    be captured in a CUDA graph when no eager autograd graph of the same table is alive.
    """
    if table.is_cuda:
        return _C.embedding_lookup(table, idx, scale, table_sf)          # (which looks at every argument, and is the autograd node)
    assert table.dim() == 2 and idx.dtype in (torch.int64, torch.int32), 'table [rows, hidden], idx int64 or int32'
    assert idx.device == table.device, 'table and indices lie on one device'
    if table_sf is not None:
        assert table.dtype == torch.float8_e4m3fn and table_sf.dtype == torch.float32 and table.size(1) % 128 == 0, \
            'scales belong to an e4m3 table whose width is a multiple of 128'
        assert table_sf.shape == (table.size(0), table.size(1) // 128), 'one scale per row and 128 columns'
        return _lookup(table.detach(), idx, float(scale), table_sf.detach())
    assert table.dtype in _TABLE_TYPES, 'the table is bf16, fp16 or fp32, or e4m3 with `table_sf`'
    if not (torch.is_grad_enabled() and table.requires_grad):
        return _lookup(table, idx, float(scale), None)
    return _Lookup.apply(table, idx, float(scale))


def embedding_grad(dy: torch.Tensor, idx: torch.Tensor, num_rows: int, scale: float = 1.0,
                   out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """Gradient of `embedding_lookup` in the table: `out[v] = scale * sum of dy[t] over idx[t] == v`, `[num_rows, hidden]`.

    `dy` is `[idx.numel(), hidden]` (bf16, fp16 or fp32). The result has its type, or is written to `out` (that type or fp32;
    rows without a token become zero). With `accumulate` the sums are added to an fp32 `out` instead, and only the rows of
    tokens are touched. Sums are in fp32, in token order, scaled and rounded once.
    """
    if dy.is_cuda:
        return _C.embedding_grad(dy, idx, num_rows, scale, out, accumulate)          # (which looks at every argument)
    assert dy.dim() == 2 and dy.size(0) == idx.numel() and dy.dtype in _TABLE_TYPES, 'dy is [number of indices, hidden]'
    assert idx.dtype in (torch.int64, torch.int32) and idx.device == dy.device
    assert num_rows >= 0
    if out is None:
        assert not accumulate, 'accumulation needs `out`'
        out = torch.empty((num_rows, dy.size(1)), dtype=dy.dtype, device=dy.device)
    assert out.shape == (num_rows, dy.size(1)) and out.device == dy.device, 'out is [num_rows, hidden]'
    assert out.dtype == torch.float32 or (out.dtype == dy.dtype and not accumulate), 'out is fp32, or of dy\'s type and overwritten'
    flat = idx.reshape(-1)
    valid = (flat >= 0) & (flat < num_rows)
    sums = torch.zeros((num_rows, dy.size(1)), dtype=torch.float32).index_add_(0, flat[valid].long(), dy[valid].float()) * scale
    with torch.no_grad():
        return out.add_(sums) if accumulate else out.copy_(sums)
