"""The longest batches with gradients of A and B, and the first that is too long: refused by the forward pass, not by the backward one."""
import pytest
import torch

from deep_ep.ops.lora import lora_linear

MOST = 2 ** 23


def make(rows):
    gen = torch.Generator(device='cuda').manual_seed(1)
    draw = lambda *s: torch.randint(-1, 2, s, generator=gen, device='cuda').to(torch.bfloat16)          # noqa: E731
    return draw(rows, 8), draw(8, 8), draw(2, 8, 8), draw(2, 8, 8), draw(rows, 8), torch.randint(-1, 2, (rows,), generator=gen, device='cuda', dtype=torch.int32)


@pytest.mark.gpu
def test_as_many_rows_as_fit():
    """Operands of -1, 0 and 1: t, and the sums over the rows, are whole numbers far below 2^24 and exact in fp32."""
    x, w, a, b, dy, idx = make(MOST)
    for t in (a, b):
        t.requires_grad_()
        t.main_grad = torch.zeros_like(t, dtype=torch.float32)
    lora_linear(x, w, a, b, idx).backward(dy)
    for e in range(2):
        mine = (idx == e).double().unsqueeze(1)
        t, dt = (x.double() @ a[e].detach().double().t()) * mine, (dy.double() @ b[e].detach().double()) * mine
        assert torch.equal(a.main_grad[e].double(), dt.t() @ x.double()) and torch.equal(b.main_grad[e].double(), dy.double().t() @ t)


@pytest.mark.gpu
def test_one_row_more():
    import deep_ep
    x, w, a, b, dy, idx = make(MOST + 1)
    with torch.no_grad():
        y = lora_linear(x, w, a.requires_grad_(), b, idx)
    assert y.shape == (MOST + 1, 8)
    with pytest.raises(deep_ep.EPException, match='rows'):
        lora_linear(x, w, a, b, idx)
    a.requires_grad_(False)
    x.requires_grad_()
    dx, = torch.autograd.grad(lora_linear(x, w, a, b, idx), x, dy)
    last = slice(MOST - 200, MOST + 1)
    want = dy[last].double() @ w.double()
    for e in range(2):
        want += (idx[last] == e).double().unsqueeze(1) * (dy[last].double() @ b[e].double() @ a[e].double())
    assert torch.equal(dx[last].double(), want.to(torch.bfloat16).double())
