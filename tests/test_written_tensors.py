"""Tensors that the operators write into count as modified, as they do after a torch operation in place: a graph that has saved
one of them refuses to go back through it."""
import pytest
import torch

from deep_ep.ops.embedding import embedding_grad, embedding_lookup
from deep_ep.ops.grad_norm import clip_grad_norm_, grad_norm
from deep_ep.ops.lora import lora_linear
from test_lora import make

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def versions(tensors):
    return [t._version for t in tensors]


@pytest.mark.parametrize('device', DEVICES)
def test_clipping(device):
    grads = [torch.ones(100, device=device), torch.ones(33, device=device, dtype=torch.bfloat16), torch.ones(0, device=device)]
    before = versions(grads)
    grad_norm(grads)
    assert versions(grads) == before
    out = [torch.empty_like(g) for g in grads]
    out_before = versions(out)
    clip_grad_norm_(grads, 1.0, out=out)
    assert versions(grads) == before and all(v > o for v, o in zip(versions(out)[:2], out_before))
    clip_grad_norm_(grads[1:], 1.0, replicated=grads[:1])
    assert all(v > o for v, o in zip(versions(grads)[:2], before))


@pytest.mark.parametrize('device', DEVICES)
def test_a_graph_that_saved_a_clipped_tensor(device):
    leaf = torch.ones(10, device=device, requires_grad=True)
    g = leaf * 3
    y = (g * g).sum()
    clip_grad_norm_([g.detach()], 1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


@pytest.mark.parametrize('device', DEVICES)
def test_embedding_gradient(device):
    dy, ids = torch.ones(5, 8, device=device), torch.tensor([0, 1, 1, -1, 3], device=device)
    whole = torch.zeros(8, 8, device=device)
    for out, accumulate, rows in ((whole[:4], False, 5), (whole[2:6], True, 5), (whole[:4], False, 0)):          # (a view counts for what it views)
        before = whole._version
        embedding_grad(dy[:rows], ids[:rows], 4, out=out, accumulate=accumulate)
        assert whole._version > before


@pytest.mark.parametrize('device', DEVICES)
def test_main_grad_of_tables(device):
    table = torch.ones(4, 8, device=device, requires_grad=True)
    table.main_grad = torch.zeros(4, 8, device=device)
    before = table.main_grad._version
    embedding_lookup(table, torch.tensor([0, 1, 1], device=device)).sum().backward()
    assert table.main_grad._version > before and table.main_grad[1, 0] == 2


@pytest.mark.parametrize('device', DEVICES)
def test_main_grad_of_adapters(device):
    x, w, a, b, dy, idx, s = make(20, 64, 32, 8, 2, device)
    for t in (a, b):
        t.requires_grad_()
        t.main_grad = torch.zeros_like(t, dtype=torch.float32)
    before = versions([a.main_grad, b.main_grad])
    lora_linear(x, w, a, b, idx, s).backward(dy)
    assert all(v > o for v, o in zip(versions([a.main_grad, b.main_grad]), before)) and a.main_grad.any()


@pytest.mark.gpu
def test_inference_tensors_are_still_written():
    with torch.inference_mode():
        g, out = torch.full((100,), 2.0, device='cuda'), torch.zeros(4, 8, device='cuda')
        clip_grad_norm_([g], 10.0)
    assert abs(float(clip_grad_norm_([g], 10.0)) - 10) < 1e-5
    embedding_grad(torch.ones(2, 8, device='cuda'), torch.tensor([1, 1], device='cuda'), 4, out=out)
    assert out[1, 0] == 2
