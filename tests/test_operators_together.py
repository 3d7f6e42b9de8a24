"""The operators around the MoE layer as a fine-tuning step runs them: token ids -> scaled embedding -> shared projection with
adapters -> MoE layer -> backward -> global norm and clipping, and what a serving step runs of them."""
import math

import pytest
import torch
import torch.distributed as dist

from deep_ep.ops.embedding import embedding_lookup
from deep_ep.ops.grad_norm import clip_grad_norm_
from deep_ep.ops.lora import lora_linear
from dist_utils import run_distributed


def _step_worker(rank, world, device):
    """One step on every rank; each operator's gradient is checked against the formula at the gradient that reached it."""
    from deep_ep.models.moe_layer import MoEConfig, MoELayer
    torch.manual_seed(3)
    tokens, vocab, hidden, rank_r, adapters = 96, 300, 128, 8, 3
    cfg = MoEConfig(hidden=hidden, intermediate=128, num_experts=8 if device == 'cpu' else 128, num_topk=2, num_shared_experts=1,
                    num_max_tokens_per_rank=tokens, expert_alignment=16 if device == 'cpu' else 128,
                    expert_backend='torch' if device == 'cpu' else 'grouped')
    table = (torch.randn(vocab, hidden, device=device) * 0.1).to(torch.bfloat16).requires_grad_()
    w = (torch.randn(hidden, hidden, device=device) * hidden ** -0.5).to(torch.bfloat16)
    a = (torch.randn(adapters, rank_r, hidden, device=device) * hidden ** -0.5).to(torch.bfloat16).requires_grad_()
    b = (torch.randn(adapters, hidden, rank_r, device=device) * 0.3).to(torch.bfloat16).requires_grad_()
    layer = MoELayer(dist.group.WORLD, cfg, device=torch.device(device))
    assert float(layer.clip_grad_norm_(1.0)) == 0.0                  # no gradients yet
    torch.manual_seed(10 + rank)
    ids = torch.randint(-1, vocab, (tokens,), device=device)
    idx = torch.randint(-1, adapters, (tokens,), device=device)
    e = embedding_lookup(table, ids, math.sqrt(hidden))
    h = lora_linear(e, w, a, b, idx, 2.0)
    kept = {}
    e.register_hook(lambda g: kept.__setitem__('e', g.clone()))
    h.register_hook(lambda g: kept.__setitem__('h', g.clone()))
    layer(h).float().square().mean().backward()

    # gradients of the operators, from the gradients that arrived at them
    f64 = torch.float64
    de, dh, ed = kept['e'].to(f64), kept['h'].to(f64), e.detach().to(f64)
    expected = torch.zeros(vocab, hidden, dtype=f64, device=device).index_add_(0, ids.clamp(min=0), de * (ids >= 0).unsqueeze(1)) * math.sqrt(hidden)
    near = lambda got, want: assert_near(got.to(f64), want)          # noqa: E731
    near(table.grad, expected)
    da, db, dx = torch.zeros_like(a, dtype=f64), torch.zeros_like(b, dtype=f64), dh @ w.to(f64)
    for n in range(adapters):
        rows = torch.nonzero(idx == n).flatten()
        t, dt = 2.0 * ed[rows] @ a.detach()[n].to(f64).t(), 2.0 * dh[rows] @ b.detach()[n].to(f64)
        da[n], db[n] = dt.t() @ ed[rows], dh[rows].t() @ t
        dx[rows] += dt @ a.detach()[n].to(f64)
    near(a.grad, da), near(b.grad, db), near(kept['e'], dx)

    # the norm over everything: what every rank holds is averaged first and counts once, the experts' gradients differ by rank
    replicated = [table, a, b, layer.gate, layer.shared_gate_up, layer.shared_down]
    if world > 1:
        for p in replicated:
            mean = p.grad.float()
            dist.all_reduce(mean)
            p.grad.copy_(mean / world)
    experts = [layer.w_gate_up.grad, layer.w_down.grad]
    squares = torch.stack([g.double().square().sum() for g in experts]).sum()
    if world > 1:
        dist.all_reduce(squares)
    ref = math.sqrt(float(squares) + sum(float(p.grad.double().square().sum()) for p in replicated))
    grads = experts + [p.grad for p in replicated]
    before = [g.clone() for g in grads]
    norm = clip_grad_norm_(experts, ref / 2, group=dist.group.WORLD if world > 1 else None, replicated=[p.grad for p in replicated])
    assert abs(float(norm) - ref) <= 1e-6 * ref
    for g, o in zip(grads, before):
        assert torch.allclose(g.double(), o.double() * 0.5, rtol=2.0 ** -8, atol=1e-30)
    # the layer's own clipping, at a limit that is not reached: the same norm of its part, nothing changed
    part = [layer.gate, layer.shared_gate_up, layer.shared_down]
    squares = torch.stack([g.double().square().sum() for g in experts]).sum()
    if world > 1:
        dist.all_reduce(squares)
    ref = math.sqrt(float(squares) + sum(float(p.grad.double().square().sum()) for p in part))
    kept_grads = [g.clone() for g in grads]
    assert abs(float(layer.clip_grad_norm_(ref * 2)) - ref) <= 1e-6 * ref
    assert all(torch.equal(g, k) for g, k in zip(grads, kept_grads))
    layer.destroy()


def assert_near(got, want):
    """One rounding to bf16 (2^-8 of the value) and, below it, 2^-12 of the largest for the fp32 sums and bf16 halves."""
    assert ((got - want).abs() <= want.abs() * 2.0 ** -8 + want.abs().max() * 2.0 ** -12).all()


@pytest.mark.parametrize('world', [1, 2])
def test_training_step_on_cpu_ranks(world, master_port):
    run_distributed(_step_worker, world, master_port, 'gloo', args=('cpu',), timeout_s=180)


@pytest.mark.gpu
def test_training_step_on_the_gpu(master_port):
    run_distributed(_step_worker, 1, master_port, 'nccl', args=('cuda',), timeout_s=180)


@pytest.mark.gpu
def test_captured_training_steps():
    """Forward, backward, clipping and update in one CUDA graph, replayed on other batches, against the same steps run eagerly."""
    def make():
        torch.manual_seed(0)
        table = (torch.randn(500, 256, device='cuda') * 0.1).to(torch.bfloat16)
        w = (torch.randn(128, 256, device='cuda') * 0.06).to(torch.bfloat16)
        a, b = (torch.randn(4, 16, 256, device='cuda') * 0.06).to(torch.bfloat16), torch.zeros(4, 128, 16, device='cuda', dtype=torch.bfloat16)
        leaves = [t.requires_grad_() for t in (table, a, b)]
        for t in leaves:
            t.main_grad = torch.zeros_like(t, dtype=torch.float32)
        return leaves, w

    def step(leaves, w, ids, idx, target):
        for t in leaves:
            t.main_grad.zero_()
        y = lora_linear(embedding_lookup(leaves[0], ids, 16.0), w, leaves[1], leaves[2], idx, 0.5)
        (y.float() - target).square().sum().backward()
        norm = clip_grad_norm_([t.main_grad for t in leaves], 1.0)
        with torch.no_grad():
            for t in leaves:
                t.add_(t.main_grad, alpha=-0.5)
        return norm

    batches = []
    for seed in range(4):
        torch.manual_seed(seed)
        batches.append((torch.randint(-1, 500, (300,), device='cuda'), torch.randint(-1, 4, (300,), device='cuda'),
                        torch.randn(300, 128, device='cuda')))
    eager, w = make()
    norms = [step(eager, w, *batch) for batch in batches]
    captured, w = make()
    static = [t.clone() for t in batches[0]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        saved = [t.detach().clone() for t in captured]
        step(captured, w, *static)                  # warm-up, taken back
        with torch.no_grad():
            for t, s in zip(captured, saved):
                t.copy_(s)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step(captured, w, *static)
    for batch, want in zip(batches, norms):
        for s, t in zip(static, batch):
            s.copy_(t)
        graph.replay()
        assert torch.equal(norm, want)
    for got, want in zip(captured, eager):
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize('tokens', [1, 33, 128])
def test_serving_step(tokens):
    """Decode: 8-bit entry rows, then two projections with adapters whose indices differ from row to row."""
    torch.manual_seed(tokens)
    entries = (torch.randn(1000, 512, device='cuda') * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    sf = torch.rand(1000, 4, device='cuda') * 0.02
    w1, w2 = (torch.randn(1024, 512, device='cuda') * 0.04).bfloat16(), (torch.randn(512, 1024, device='cuda') * 0.03).bfloat16()
    make = lambda e, n, k: (torch.randn(e, n, k, device='cuda') * k ** -0.5).bfloat16()            # noqa: E731
    a1, b1, a2, b2 = make(20, 16, 512), make(20, 1024, 16), make(20, 16, 1024), make(20, 512, 16)
    ids, idx = torch.randint(0, 1000, (tokens,), device='cuda'), torch.randint(-1, 20, (tokens,), device='cuda', dtype=torch.int32)
    with torch.no_grad():
        x = embedding_lookup(entries, ids, 1.0, table_sf=sf)
        h = lora_linear(x, w1, a1, b1, idx)
        y = lora_linear(h, w2, a2, b2, idx)

    def reference(x, w, a, b):
        x = x.double()
        out = x @ w.double().t()
        for e in range(20):
            rows = torch.nonzero(idx == e).flatten()
            out[rows] += (x[rows] @ a[e].double().t()) @ b[e].double().t()
        return out
    expected = entries[:, :].float().double()[ids] * sf.double()[ids].repeat_interleave(128, dim=1)
    assert ((x.double() - expected).abs() <= expected.abs() * 2.0 ** -8 * 1.001).all()
    assert_near(h.double(), reference(x, w1, a1, b1))
    assert_near(y.double(), reference(h, w2, a2, b2))
