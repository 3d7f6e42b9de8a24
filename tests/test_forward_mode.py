"""Forward-mode differentiation: the CPU forms carry tangents, the kernels do not and refuse a tensor that has one."""
import pytest
import torch
from torch.autograd import forward_ad

from deep_ep.ops.embedding import embedding_grad, embedding_lookup
from deep_ep.ops.grad_norm import clip_grad_norm_, grad_norm
from deep_ep.ops.lora import lora_linear
from test_lora import make


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def test_cpu_forms_carry_tangents():
    table, ids = torch.randn(9, 16), torch.tensor([3, -1, 3])
    x, w, a, b, dy, idx, s = make(9, 16, 8, 8, 2, 'cpu')
    with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(embedding_lookup(dual(table), ids, 2.0)).tangent
        assert torch.equal(tangent, torch.tensor([2.0, 0.0, 2.0]).unsqueeze(1).expand(3, 16))
        for i in range(4):
            args = [x, w, a, b]
            args[i] = dual(args[i])
            assert forward_ad.unpack_dual(lora_linear(*args, idx, s)).tangent.any()


@pytest.mark.gpu
@pytest.mark.parametrize('wanted', [False, True], ids=['without gradients', 'with gradients'])
def test_kernels_refuse_tangents(wanted):
    import deep_ep
    table, ids = torch.randn(9, 16, device='cuda').requires_grad_(wanted), torch.tensor([3, -1, 3], device='cuda')
    rows, out = torch.randn(3, 16, device='cuda'), torch.zeros(9, 16, device='cuda')
    x, w, a, b, dy, idx, s = make(9, 128, 128, 8, 2, 'cuda')
    operands = [t.requires_grad_(wanted) for t in (x, w, a, b)]
    with forward_ad.dual_level():
        with pytest.raises(deep_ep.EPException, match='forward-mode'):
            embedding_lookup(dual(table), ids, 2.0)
        for i in range(4):
            args = [dual(t) if i == j else t for j, t in enumerate(operands)]
            with pytest.raises(deep_ep.EPException, match='forward-mode'):
                lora_linear(*args, idx, s)
        for bad in (lambda: lora_linear(*operands, idx, dual(s)), lambda: embedding_grad(dual(rows), ids, 9), lambda: embedding_grad(rows, ids, 9, out=dual(out)),
                    lambda: clip_grad_norm_([dual(rows)], 1.0), lambda: clip_grad_norm_([rows, out], 1.0, out=[rows, dual(out)])):
            with pytest.raises(deep_ep.EPException, match='forward-mode'):
                bad()
        # tensors without a tangent, and a norm, which carries no derivative on the CPU either
        assert embedding_lookup(table, ids).shape == (3, 16) and lora_linear(*operands, idx, s).shape == (9, 128)
        assert forward_ad.unpack_dual(grad_norm([dual(rows)])).tangent is None
    assert embedding_lookup(table, ids).shape == (3, 16)
