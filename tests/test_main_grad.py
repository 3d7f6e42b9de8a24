"""Weight gradients that go to a parameter's fp32 `main_grad` buffer: on the CPU as on the GPU, also when the forward pass is
checkpointed or its saved tensors are stored elsewhere (a hook hands the backward pass other tensors than the parameters then),
and clipping of a layer whose parameters carry such buffers."""
import math

import pytest
import torch
import torch.distributed as dist
from torch.utils.checkpoint import checkpoint

from deep_ep.ops.embedding import embedding_lookup
from deep_ep.ops.lora import lora_linear
from dist_utils import run_distributed
from test_grouped_gemm_gpu import make_layout
from test_lora import U, check, make, reference

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def test_adapters_on_the_cpu():
    x, w, a, b, dy, idx, s = make(37, 48, 24, 6, 3, 'cpu')
    leaves = [t.clone().requires_grad_() for t in (w, a, b)]
    for t in leaves[1:]:
        t.main_grad = torch.zeros_like(t, dtype=torch.float32)
    for _ in range(2):
        lora_linear(x, *leaves, idx, s).backward(dy)
    assert leaves[1].grad is None and leaves[2].grad is None and leaves[0].grad is not None
    refs, bounds = reference(x, w, a, b, dy, idx, s)
    check(leaves[1].main_grad, 2 * refs[2], 2 * bounds[2], 2 * U)
    check(leaves[2].main_grad, 2 * refs[3], 2 * bounds[3], 2 * U)


@pytest.mark.parametrize('device', DEVICES)
def test_one_adapter_matrix_with_a_buffer(device):
    """A with a buffer, B without: each where it belongs, and the same bits as without any."""
    x, w, a, b, dy, idx, s = make(50, 64, 32, 8, 3, device)
    plain = [t.clone().requires_grad_() for t in (x, a, b)]
    y = lora_linear(plain[0], w, plain[1], plain[2], idx, s)
    y.backward(dy)
    mixed = [t.clone().requires_grad_() for t in (x, a, b)]
    mixed[1].main_grad = torch.zeros_like(a, dtype=torch.float32)
    z = lora_linear(mixed[0], w, mixed[1], mixed[2], idx, s)
    z.backward(dy)
    assert torch.equal(y, z) and torch.equal(plain[0].grad, mixed[0].grad) and torch.equal(plain[2].grad, mixed[2].grad)
    assert mixed[1].grad is None and torch.equal(mixed[1].main_grad.to(torch.bfloat16), plain[1].grad)


def test_cpu_adapters_without_a_buffer_can_be_differentiated_twice_and_forward():
    x, w, a, b, dy, idx, s = make(9, 16, 8, 8, 2, 'cpu')
    leaves = [t.clone().requires_grad_() for t in (a, b)]
    y = lora_linear(x, w, *leaves, idx, s)
    da, = torch.autograd.grad(y, leaves[0], dy, create_graph=True)
    assert torch.autograd.grad(da.float().square().sum(), leaves[1])[0].any()
    with torch.autograd.forward_ad.dual_level():
        y = lora_linear(x, w, torch.autograd.forward_ad.make_dual(a, torch.ones_like(a)), b, idx, s)
        assert torch.autograd.forward_ad.unpack_dual(y).tangent.any()


# ------------------------------------------------------------------------------------------------ hooks on saved tensors
def embedding_case(device):
    table = torch.randn(50, 16, device=device).to(torch.bfloat16)
    ids, dy = torch.randint(0, 50, (40,), device=device), torch.randn(40, 16, device=device).to(torch.bfloat16)
    return [table], lambda p: embedding_lookup(p[0], ids, 2.0), dy


def adapter_case(device):
    x, w, a, b, dy, idx, s = make(150, 64, 128, 16, 3, device)
    return [a, b], lambda p: lora_linear(x, w, p[0], p[1], idx, s), dy


def grouped_linear_case(device):
    from deep_ep.ops.grouped_gemm import GroupedLinear
    psum, count, rows, _ = make_layout([100, 0, 37], 128, torch.device(device))
    x, w = torch.randn(rows, 256, device=device).to(torch.bfloat16), (torch.randn(3, 128, 256, device=device) * 0.06).to(torch.bfloat16)
    dy = torch.randn(rows, 128, device=device).to(torch.bfloat16)
    return [w], lambda p: GroupedLinear.apply(x, p[0], psum, count, 128), dy


def ffn_case(device, fp8):
    from deep_ep.ops.fp8_training import Fp8WeightCache, grouped_swiglu_ffn_fp8_training
    from deep_ep.ops.grouped_gemm import grouped_swiglu_ffn
    psum, count, rows, starts = make_layout([100, 0, 37], 128, torch.device(device))
    x, dy = (torch.zeros(rows, 512, dtype=torch.bfloat16, device=device) for _ in range(2))
    for start, c in zip(starts, [100, 0, 37]):
        x[start:start + c], dy[start:start + c] = torch.randn(c, 512).to(device), torch.randn(c, 512).to(device)
    w1, w2 = ((torch.randn(*shape) * 0.05).to(torch.bfloat16).to(device) for shape in ((3, 1024, 512), (3, 512, 512)))
    cache = Fp8WeightCache()
    if fp8:
        return [w1, w2], lambda p: grouped_swiglu_ffn_fp8_training(x, *p, psum, count, 128, cache), dy
    return [w1, w2], lambda p: grouped_swiglu_ffn(x, *p, psum, count, None, 128), dy


CASES = [('cpu', embedding_case, ()), ('cpu', adapter_case, ()), ('cpu', ffn_case, (True,))] + [
    pytest.param('cuda', *c, marks=pytest.mark.gpu) for c in ((embedding_case, ()), (adapter_case, ()), (grouped_linear_case, ()),
                                                              (ffn_case, (False,)), (ffn_case, (True,)))]


@pytest.mark.parametrize('how', ['checkpoint', 'hooks'])
@pytest.mark.parametrize('device,case,args', CASES)
def test_under_saved_tensor_hooks(device, case, args, how):
    torch.manual_seed(0)
    values, forward, dy = case(device, *args)

    def run(wrapped):
        leaves = [v.clone().requires_grad_() for v in values]
        for t in leaves:
            t.main_grad = torch.zeros_like(t, dtype=torch.float32)
        if not wrapped:
            y = forward(leaves)
        elif how == 'checkpoint':
            y = checkpoint(lambda *p: forward(p), *leaves, use_reentrant=False)
        else:
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t):
                y = forward(leaves)
        y.backward(dy)
        assert all(t.grad is None for t in leaves)
        return [t.main_grad for t in leaves]

    for plain, hooked in zip(run(False), run(True)):
        assert plain.any() and torch.equal(plain, hooked)


# ------------------------------------------------------------------------------------------------ the layer's clipping
def _clip_worker(rank, world, device):
    from deep_ep.models.moe_layer import MoEConfig, MoELayer
    torch.manual_seed(3)
    cfg = MoEConfig(hidden=128, intermediate=128, num_experts=8 if device == 'cpu' else 128, num_topk=2, num_shared_experts=1,
                    num_max_tokens_per_rank=64, expert_alignment=16 if device == 'cpu' else 128,
                    expert_backend='torch' if device == 'cpu' else 'grouped')
    layer = MoELayer(dist.group.WORLD, cfg, device=torch.device(device))
    experts, others = [layer.w_gate_up, layer.w_down], [layer.gate, layer.shared_gate_up, layer.shared_down]

    def step(stale):
        """Gradients of one step, every parameter with a buffer; those that no kernel adds to hold `stale`."""
        for p in experts + others:
            p.grad, p.main_grad = None, torch.full_like(p, 0.0 if p is layer.w_gate_up or p is layer.w_down else stale, dtype=torch.float32)
        torch.manual_seed(10 + rank)
        layer(torch.randn(64, 128, device=device).to(torch.bfloat16)).float().square().mean().backward()

    def norm_of(sharded, replicated):
        squares = torch.stack([g.double().square().sum() for g in sharded]).sum()
        if world > 1:
            dist.all_reduce(squares)
        return math.sqrt(float(squares) + sum(float(g.double().square().sum()) for g in replicated))

    def clipped(grads, call, ref):
        before = [g.clone() for g in grads]
        assert abs(float(call()) - ref) <= 1e-6 * ref
        for g, o in zip(grads, before):
            assert o.any() and torch.allclose(g.double(), o.double() * (ref / 2 / (ref + 1e-6)), rtol=torch.finfo(g.dtype).eps + 1e-6, atol=1e-30)

    step(1e3)
    for p in others:
        assert p.grad is not None
        if world > 1:
            mean = p.grad.float()
            dist.all_reduce(mean)
            p.grad.copy_(mean / world)
    # the kernels add the experts' gradients to their buffers, plain torch operations leave them in `.grad`
    held = [p.grad if device == 'cpu' else p.main_grad for p in experts]
    assert all((p.grad is None) == (device != 'cpu') for p in experts)
    plain = [p.grad for p in others]
    ref = norm_of(held, plain)
    clipped(held + plain, lambda: layer.clip_grad_norm_(ref / 2), ref)
    assert all((p.main_grad == 1e3).all() for p in others)
    # a training loop that moves every gradient into its buffer
    step(0.0)
    for p in experts + others:
        if p.grad is not None:
            p.main_grad.add_(p.grad)
            p.grad = None
    if world > 1:
        for p in others:
            dist.all_reduce(p.main_grad)
    ref = norm_of([p.main_grad for p in experts], [p.main_grad for p in others])
    clipped([p.main_grad for p in experts + others], lambda: layer.clip_grad_norm_(ref / 2), ref)
    layer.destroy()


@pytest.mark.parametrize('world', [1, 2])
def test_layer_clipping_with_buffers_on_cpu_ranks(world, master_port):
    run_distributed(_clip_worker, world, master_port, 'gloo', args=('cpu',), timeout_s=180)


@pytest.mark.gpu
def test_layer_clipping_with_buffers_on_the_gpu(master_port):
    run_distributed(_clip_worker, 1, master_port, 'nccl', args=('cuda',), timeout_s=180)
