"""Infinities and NaN in adapters, rows and gradients: every element of every result has the class (finite, +inf, -inf, NaN) that
the formulas give in 64 bits, whatever kernel a call takes and whichever requests share its tiles.

A product t * inf has the sign of t, so the class of an element is certain where t is larger than the error of its sum in
fp32, (k + 1) * 2^-23 of the sum of magnitudes: rows of the checked adapter where it is not are left out."""
import pytest
import torch

from deep_ep.ops.lora import lora_linear
from test_lora import BF16, U, make

INF, NAN = float('inf'), float('nan')
# rows, K, N, rank. One row tile with few elements of t; a cluster that shares a tile; single CTAs with several tiles each, in the
# forward and in the backward product; pairs of CTAs in both
GPU_SHAPES = [(20, 512, 256, 8), (100, 512, 256, 40), (384, 64, 9728, 40), (384, 9728, 64, 40), (700, 256, 8192, 40), (700, 8192, 256, 40)]
CASES = [('cpu', (20, 64, 48, 8)), ('cpu', (37, 32, 72, 40))] + [pytest.param('cuda', shape, marks=pytest.mark.gpu) for shape in GPU_SHAPES]


def classes(t):
    return torch.where(t.isnan(), 3, torch.where(t == INF, 1, torch.where(t == -INF, 2, 0)))


def formulas(x, w, a, b, dy, idx, s):
    """y, dx, dA, dB in 64 bits, and t, dt."""
    x, w, a, b, dy, s, idx = (v.detach().double() if v.is_floating_point() else v for v in (x, w, a, b, dy, s, idx))
    y, dx, da, db = x @ w.t(), dy @ w, torch.zeros_like(a), torch.zeros_like(b)
    t, dt = x.new_zeros(x.size(0), a.size(1)), x.new_zeros(x.size(0), a.size(1))
    for e in range(a.size(0)):
        at = torch.nonzero(idx == e).flatten()
        t[at], dt[at] = s[e] * (x[at] @ a[e].t()), s[e] * (dy[at] @ b[e])
        y[at] += t[at] @ b[e].t()
        dx[at] += dt[at] @ a[e]
        da[e], db[e] = dt[at].t() @ x[at], dy[at].t() @ t[at]
    return y, dx, da, db, t, dt


def certain(t, left, right, s):
    """t = s * left . right^T, elements whose sign survives fp32."""
    return t.abs() > s * (left.double().abs() @ right.double().abs().t()) * (left.size(1) + 1) * U


def run(x, w, a, b, dy, idx, s):
    leaves = [v.detach().clone().requires_grad_() for v in (x, a, b)]
    y = lora_linear(leaves[0], w, leaves[1], leaves[2], idx, s)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def problem(shape, order, device, seed=4):
    x, w, a, b, dy, idx, s = make(*shape, 3, device, order, seed=seed)
    if order == 'mixed':
        idx = torch.where(torch.arange(idx.numel(), device=device) < 3, torch.arange(idx.numel(), device=device, dtype=idx.dtype) % 3, idx)
    return x, w, a, b, dy, idx, s


def near(got, want):
    """Finite elements: one rounding, and 2^-12 of the largest for the fp32 sums."""
    finite = want.isfinite()
    assert ((got.double() - want)[finite].abs() <= want[finite].abs() * BF16 + want[finite].abs().max() * 2.0 ** -12).all()


@pytest.mark.parametrize('device,shape', CASES, ids=str)
@pytest.mark.parametrize('order', ['same', 'mixed'])
def test_bad_adapters(device, order, shape):
    x, w, a, b, dy, idx, s = problem(shape, order, device)
    e = 2
    rows = torch.nonzero(idx == e).flatten()
    # B: single infinities of both signs, two in one column, a NaN; next to finite elements in the same 16 bytes
    bad = b.clone()
    bad[e, 5, 3], bad[e, 11, 3], bad[e, 17, 2], bad[e, 17, 5], bad[e, 20, 1] = INF, -INF, INF, INF, NAN
    want = formulas(x, w, a, bad, dy, idx, s)
    sure = certain(want[4][rows], x[rows], a[e], s[e].item())[:, [2, 3, 5]].all(dim=1)
    assert sure.sum() > 0
    y = lora_linear(x, w, a, bad, idx, s)
    keep = torch.ones(x.size(0), dtype=torch.bool, device=device)
    keep[rows[~sure]] = False
    assert torch.equal(classes(y)[keep], classes(want[0])[keep])
    near(y, want[0])
    # A, in the data gradient
    bad = a.clone()
    bad[e, 3, 5], bad[e, 3, 11], bad[e, 2, 17], bad[e, 5, 17], bad[e, 1, 20] = INF, -INF, INF, INF, NAN
    want = formulas(x, w, bad, b, dy, idx, s)
    sure = certain(want[5][rows], dy[rows], b[e].t(), s[e].item())[:, [2, 3, 5]].all(dim=1)
    assert sure.sum() > 0
    dx = run(x, w, bad, b, dy, idx, s)[1]
    keep = torch.ones(x.size(0), dtype=torch.bool, device=device)
    keep[rows[~sure]] = False
    assert torch.equal(classes(dx)[keep], classes(want[1])[keep])
    near(dx, want[1])


@pytest.mark.parametrize('device,shape', CASES, ids=str)
@pytest.mark.parametrize('order', ['same', 'mixed'])
@pytest.mark.parametrize('value', [INF, -INF, NAN], ids=str)
def test_bad_rows(device, order, shape, value):
    """One element of one row of x, then of dy: results of the row, and gradients of its adapter."""
    x, w, a, b, dy, idx, s = problem(shape, order, device)
    e = 2
    row = int(torch.nonzero(idx == e)[0])
    clean = formulas(x, w, a, b, dy, idx, s)
    sure_t = certain(clean[4][[row]], x[[row]], a[e], s[e].item())[0]
    sure_dt = certain(clean[5][[row]], dy[[row]], b[e].t(), s[e].item())[0]
    bad = x.clone()
    bad[row, 9] = value
    want = formulas(bad, w, a, b, dy, idx, s)
    got = run(bad, w, a, b, dy, idx, s)
    for i in (0, 1, 3):
        assert torch.equal(classes(got[i]), classes(want[i])), i
    assert torch.equal(classes(got[2])[:, sure_dt], classes(want[2])[:, sure_dt])
    bad = dy.clone()
    bad[row, 9] = value
    want = formulas(x, w, a, b, bad, idx, s)
    got = run(x, w, a, b, bad, idx, s)
    for i in (0, 1, 2):
        assert torch.equal(classes(got[i]), classes(want[i])), i
    assert torch.equal(classes(got[3])[:, :, sure_t], classes(want[3])[:, :, sure_t])


@pytest.mark.parametrize('device,shape', CASES, ids=str)
@pytest.mark.parametrize('order', ['same', 'mixed'])
def test_bad_row_of_a_bad_adapter(device, order, shape):
    """Infinities on both sides of a product, whose finite neighbours in the same 16 bytes meet an infinite t. Signs are such that
    the formulas give infinities, not NaN, in some columns."""
    x, w, a, b, dy, idx, s = problem(shape, order, device)
    e = 2
    row = int(torch.nonzero(idx == e)[0])
    bad_x, bad_w, bad_a, bad_b = x.clone(), w.clone(), a.clone(), b.clone()
    bad_x[row, 9], bad_w[4:8, 9], bad_a[e, :, 9], bad_b[e, 4:8] = INF, 1, 1, b[e, 4:8].abs() + 1
    bad_b[e, 5, 3] = INF
    want = formulas(bad_x, bad_w, bad_a, bad_b, dy, idx, s)
    assert (want[0][row, 4:8] == INF).all()
    got = lora_linear(bad_x, bad_w, bad_a, bad_b, idx, s)
    assert torch.equal(classes(got)[row], classes(want[0])[row])
    bad_dy, bad_w, bad_a, bad_b = dy.clone(), w.clone(), a.clone(), b.clone()
    bad_dy[row, 9], bad_w[9, 4:8], bad_b[e, 9], bad_a[e, :, 4:8] = INF, 1, 1, a[e, :, 4:8].abs() + 1
    bad_a[e, 3, 5] = INF
    want = formulas(x, bad_w, bad_a, bad_b, bad_dy, idx, s)
    assert (want[1][row, 4:8] == INF).all()
    got = run(x, bad_w, bad_a, bad_b, bad_dy, idx, s)[1]
    assert torch.equal(classes(got)[row], classes(want[1])[row])
