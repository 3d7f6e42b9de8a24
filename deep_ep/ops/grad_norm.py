"""Global gradient norm over many tensors, and clipping by it, on hand-written kernels.

The step between the gradient reductions (`BucketBuffer.reduce_scatter` / `all_reduce`, the experts' fp32 `main_grad`
buffers) and the optimizer. Any mix of bf16, fp16 and fp32 tensors of any size and alignment; their table travels in the
launch itself, so a list of a thousand tensors takes two launches and no copy. Sums are in fp64 over short fp32 sums and in a
fixed order: the same gradients give the same bits. Nothing waits on the host, so a step can be captured in a CUDA graph.

With expert parallelism every rank holds other experts: `group` adds the squares of `grads` over its ranks. Gradients that
all ranks hold alike (router, shared expert, after their own reduction) go into `replicated` and count once.
CPU tensors take the same formulas in plain torch.
"""
from typing import List, Optional, Sequence

import torch
import torch.distributed as dist

from .._C_loader import _C

__all__ = ['grad_norm', 'clip_grad_norm_']


def _square_sums(tensors: List[torch.Tensor]) -> torch.Tensor:
    if tensors[0].is_cuda:
        return _C.grad_square_sums(tensors)
    return torch.stack([t.detach().double().square().sum() for t in tensors])


def _total(tensors: List[torch.Tensor], replicated: List[torch.Tensor], group: Optional[dist.ProcessGroup]) -> torch.Tensor:
    """fp64 tensor whose elements add up to the squared norm."""
    device = (tensors + replicated)[0].device if tensors or replicated else torch.device('cpu')
    sums = _square_sums(tensors) if tensors else torch.zeros(1, dtype=torch.float64, device=device)
    if group is not None:
        sums = sums.sum().reshape(1)
        dist.all_reduce(sums, group=group)
    if replicated:
        sums = torch.cat([sums, _square_sums(replicated)])
    return sums


def _checked(grads: Sequence[torch.Tensor], replicated: Sequence[torch.Tensor]):
    tensors, replicated = [grads] if isinstance(grads, torch.Tensor) else list(grads), list(replicated)
    everything = tensors + replicated
    if everything and everything[0].is_cuda:
        return tensors, replicated, everything         # the native call looks at types, devices and layouts, tensor by tensor
    for t in everything:
        assert t.dtype in (torch.bfloat16, torch.float16, torch.float32), 'gradients are bf16, fp16 or fp32'
        assert t.device == everything[0].device, 'gradients lie on one device'
    return tensors, replicated, everything


def grad_norm(grads: Sequence[torch.Tensor], group: Optional[dist.ProcessGroup] = None,
              replicated: Sequence[torch.Tensor] = ()) -> torch.Tensor:
    """L2 norm over all elements of all tensors as an fp32 scalar on their device (no host synchronisation).

    Tensors are dense (contiguous, or a permutation of it). With `group` the squares of `grads` are added over its ranks,
    a collective call even for a rank whose list is empty (give it a tensor in `replicated`, or an empty tensor, so that the
    device is known); `replicated` is counted once. NaN or infinity in a gradient shows in the norm."""
    if group is None and isinstance(grads, (list, tuple)) and len(grads) > 0 and grads[0].is_cuda and not replicated:
        return _C.grad_norm(grads)
    tensors, replicated, everything = _checked(grads, replicated)
    sums = _total(tensors, replicated, group)
    return _C.grad_norm_finish(sums) if sums.is_cuda else sums.sum().sqrt().float()


def clip_grad_norm_(grads: Sequence[torch.Tensor], max_norm: float, group: Optional[dist.ProcessGroup] = None,
                    replicated: Sequence[torch.Tensor] = (), out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scale `grads` and `replicated` by `min(1, max_norm / (norm + 1e-6))` in place; returns the norm before scaling.

    The product is taken in fp32 and rounded once. When the norm is within the limit nothing is written. A norm of NaN
    makes every gradient NaN, an infinite one makes finite gradients zero, as the formula says; check the returned norm.
    With `out` (one tensor per gradient, `replicated` ones last; same shapes and strides, bf16, fp16 or fp32) the scaled
    gradients are written there instead and `grads` stay as they are: fp32 accumulators become clipped bf16 gradients in
    one sweep. Tensors that are written may not share memory with one another."""
    assert max_norm >= 0, 'max_norm is not negative'
    tensors, replicated, everything = _checked(grads, replicated)
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        assert len(out) == len(everything), 'one output per gradient'
    if not everything:
        return grad_norm(tensors, group)
    if everything[0].is_cuda:
        # (without other ranks and one list, the sums are taken inside the call)
        simple = group is None and not replicated
        return _C.grad_clip(everything, out, None if simple else _total(tensors, replicated, group), float(max_norm))
    assert out is None or all(o.shape == g.shape for o, g in zip(out, everything)), 'an output has its gradient\'s shape'
    sums = _total(tensors, replicated, group)
    norm = sums.sum().sqrt().float()
    factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    with torch.no_grad():
        for o, g in zip(everything if out is None else out, everything):
            o.copy_(g.float() * factor)
    return norm
