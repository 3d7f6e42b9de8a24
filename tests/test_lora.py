"""Adapters beside a shared projection against the formulas in 64 bits.

Tolerances. bf16 products are exact in fp32; a sum of K of them on the tensor cores loses at most K * 2^-23 of the sum of
magnitudes (each addition at most 2^-23 of what is added up so far). The intermediate t = s x A^T is kept as two bf16 numbers:
2^-16 of its size. Every result is rounded to bf16 once: 2^-8 of its value. Beside that bound for each element, the whole
result is held to the size of one rounding (2^-8 in the 2-norm), which the bound's worst case would not notice."""
import pytest
import torch

from deep_ep.ops.lora import lora_linear

U = 2.0 ** -23
BF16 = 2.0 ** -8


def make(rows, k, n, rank, adapters, device, order='mixed', seed=0, none=0.15):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)          # noqa: E731
    x, w = randn(rows, k), randn(n, k) * k ** -0.5
    a, b = randn(adapters, rank, k) * k ** -0.5, randn(adapters, n, rank) * rank ** -0.5
    dy = randn(rows, n)
    idx = torch.randint(0, adapters, (rows,), generator=gen)
    if order == 'same':
        idx.fill_(adapters - 1)
    elif order == 'none':
        idx.fill_(-1)
    else:
        pick = torch.rand(rows, generator=gen)
        idx = torch.where(pick < none / 2, torch.full_like(idx, -5), torch.where(pick < none, idx + adapters, idx))
        if order == 'runs':
            idx = idx.sort().values
    scaling = torch.rand(adapters, generator=gen) + 0.5
    return [t.to(torch.bfloat16).to(device) for t in (x, w, a, b, dy)] + [idx.to(torch.int32).to(device), scaling.to(device)]


def reference(x, w, a, b, dy, idx, scaling):
    """y, dx, dA, dB in 64 bits, and for each the bound of its fp32 error."""
    x, w, a, b, dy, s = (t.detach().double() for t in (x, w, a, b, dy, scaling))
    y, dx, da, db = x @ w.t(), dy @ w, torch.zeros_like(a), torch.zeros_like(b)
    ax, aw, aa, ab, ady = x.abs(), w.abs(), a.abs(), b.abs(), dy.abs()
    k, n, r, rows = x.size(1), w.size(0), a.size(1), x.size(0)
    ey, ex, ea, eb = (ax @ aw.t()) * k * U, (ady @ aw) * n * U, torch.zeros_like(a), torch.zeros_like(b)
    for e in range(a.size(0)):
        at = torch.nonzero(idx == e).flatten()
        if at.numel() == 0:
            continue
        t, dt = s[e] * (x[at] @ a[e].t()), s[e] * (dy[at] @ b[e])
        mt, mdt = s[e] * (ax[at] @ aa[e].t()), s[e] * (ady[at] @ ab[e])
        et, edt = mt * (k + 1) * U + t.abs() * 2 ** -16, mdt * (n + 1) * U + dt.abs() * 2 ** -16
        y[at] += t @ b[e].t()
        dx[at] += dt @ a[e]
        da[e], db[e] = dt.t() @ x[at], dy[at].t() @ t
        ey[at] += et @ ab[e].t() + (t.abs() @ ab[e].t()) * (k + 2 * r) * U
        ex[at] += edt @ aa[e] + (dt.abs() @ aa[e]) * (n + 2 * r) * U
        ea[e] = edt.t() @ ax[at] + (dt.abs().t() @ ax[at]) * 2 * rows * U
        eb[e] = ady[at].t() @ et + (ady[at].t() @ t.abs()) * 2 * rows * U
    return (y, dx, da, db), (ey, ex, ea, eb)


def check(out, ref, bound, eps=BF16):
    assert out.shape == ref.shape and out.isfinite().all()
    off = (out.double() - ref).abs()
    assert (off <= ref.abs() * eps + bound).all(), f'largest excess {(off - ref.abs() * eps - bound).max()}'
    assert off.norm() <= max(eps, 2.0 ** -13) * ref.norm() + 1e-30


def run_all(args, grad=True):
    x, w, a, b, dy, idx, scaling = args
    leaves = [t.detach().clone().requires_grad_() for t in (x, a, b)]
    y = lora_linear(leaves[0], w, leaves[1], leaves[2], idx, scaling)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)] if grad else [y.detach()]


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize('order', ['mixed', 'same', 'none'])
def test_cpu_form_agrees_with_the_formulas(order):
    args = make(37, 48, 24, 6, 3, 'cpu', order)
    for out, ref, bound in zip(run_all(args), *reference(*args)):
        check(out, ref, bound)


def test_gradient_against_differences():
    """The formula's gradient itself, by differences of the plain form in 64 bits."""
    x, w, a, b, dy, idx, s = make(7, 8, 16, 8, 2, 'cpu')
    x, w, a, b, dy, s = (t.double() for t in (x, w, a, b, dy, s))

    def loss(x, a, b):
        t = torch.stack([s[e] * (x[i] @ a[e].t()) @ b[e].t() if 0 <= e < 2 else torch.zeros(16, dtype=torch.float64)
                         for i, e in enumerate(idx.tolist())])
        return ((x @ w.t() + t) * dy).sum()
    (_, dx, da, db), _ = reference(x, w, a, b, dy, idx, s)
    for value, grad in ((x, dx), (a, da), (b, db)):
        numeric = torch.zeros_like(value)
        for i in range(value.numel()):
            for sign in (1, -1):
                value.view(-1)[i] += sign * 1e-4
                numeric.view(-1)[i] += sign * loss(x, a, b) / 2e-4
                value.view(-1)[i] -= sign * 1e-4
        assert torch.allclose(numeric, grad, rtol=1e-6, atol=1e-6)


def test_refusals():
    x, w, a, b, dy, idx, s = make(5, 16, 8, 8, 2, 'cpu')
    for bad in (lambda: lora_linear(x.float(), w, a, b, idx), lambda: lora_linear(x, w[:, :8], a, b, idx), lambda: lora_linear(x, w, a, b[:, :4], idx),
                lambda: lora_linear(x, w, a, b, idx[:4]), lambda: lora_linear(x, w, a, b, idx.float()), lambda: lora_linear(x, w, a[:1], b, idx),
                lambda: lora_linear(x, w, a, b, idx, s[:1]), lambda: lora_linear(x, w, a, b, idx, s.clone().requires_grad_()),
                lambda: lora_linear(x[0], w, a, b, idx)):
        with pytest.raises(AssertionError):
            bad()


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize('rows,k,n,rank,adapters,order', [
    (1, 64, 64, 8, 1, 'same'), (1, 7168, 4096, 16, 4, 'same'), (3, 8, 8, 8, 2, 'mixed'), (130, 200, 136, 24, 5, 'mixed'),
    (127, 1000, 520, 40, 3, 'runs'), (128, 512, 256, 128, 3, 'mixed'), (96, 2048, 1024, 16, 64, 'mixed'), (300, 1024, 392, 64, 200, 'mixed'),
    (257, 640, 384, 32, 2, 'none'), (1025, 512, 2048, 48, 4, 'runs'), (2500, 1096, 2056, 72, 3, 'runs'), (5000, 256, 4096, 8, 6, 'mixed'),
    (1, 256, 128, 8, 1, 'none'), (128, 1024, 512, 32, 7, 'mixed'), (129, 1024, 512, 32, 7, 'mixed'), (500, 2048, 200, 8, 3, 'mixed'),
    (120, 4096, 1000, 64, 2, 'mixed'), (1, 128, 16384, 64, 2, 'same'), (64, 7168, 64, 128, 3, 'runs'), (700, 512, 4096, 16, 2, 'runs'),
    (19500, 64, 120, 8, 3, 'runs')])
def test_forward_and_gradients(rows, k, n, rank, adapters, order):
    args = make(rows, k, n, rank, adapters, 'cuda', order, seed=rows)
    results = run_all(args)
    for out, ref, bound in zip(results, *reference(*args)):
        check(out, ref, bound)
    again = run_all(args)
    assert all(torch.equal(p, q) for p, q in zip(results, again))
    # int64 indices, and far outside what 32 bits hold
    idx64 = args[5].long()
    idx64 = torch.where((idx64 < 0) | (idx64 >= adapters), idx64 + 2 ** 40, idx64)
    with torch.no_grad():
        assert torch.equal(lora_linear(*args[:4], idx64, args[6]), results[0])


@pytest.mark.gpu
def test_no_rows():
    x, w, a, b, dy, idx, s = make(0, 64, 128, 16, 3, 'cuda')
    y, dx, da, db = run_all((x, w, a, b, dy, idx, s))
    assert y.shape == (0, 128) and dx.shape == (0, 64) and not da.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize('rows,k,n', [(100, 512, 256), (700, 256, 8192)])
@pytest.mark.parametrize('value', [float('inf'), float('nan')], ids=str)
def test_non_finite_values_stay_with_their_request(rows, k, n, value):
    x, w, a, b, dy, idx, s = make(rows, k, n, 40, 4, 'cuda', seed=3)
    clean = run_all((x, w, a, b, dy, idx, s))
    # one bad adapter: B in one column, A in one row of another
    bad_a, bad_b = a.clone(), b.clone()
    bad_b[1, 5, 33], bad_a[2, 7, 9] = value, value
    y, dx, _, _ = run_all((x, w, bad_a, bad_b, dy, idx, s))
    others = (idx != 1) & (idx != 2)
    assert torch.equal(y[others], clean[0][others]) and torch.equal(dx[others], clean[1][others])
    one = idx == 1
    assert not y[one][:, 5].isfinite().any() and torch.equal(y[one][:, 6:], clean[0][one][:, 6:])
    assert not y[idx == 2].isfinite().any()                    # t is not finite, so no element of the row is
    assert not dx[idx == 2][:, 9].isfinite().any() and torch.equal(dx[idx == 2][:, 10:], clean[1][idx == 2][:, 10:])
    # one bad row: the others' results and the other adapters' gradients stay
    bad_x, bad_dy = x.clone(), dy.clone()
    row = int(torch.nonzero(idx == 3)[0])
    bad_x[row], bad_dy[row] = value, value
    y, dx, da, db = run_all((bad_x, w, a, b, bad_dy, idx, s))
    keep = torch.arange(rows, device='cuda') != row
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert torch.equal(da[:3], clean[2][:3]) and torch.equal(db[:3], clean[3][:3])
    assert not da[3].isfinite().all() and not db[3].isfinite().all()


@pytest.mark.gpu
def test_scaling_number_main_grad_views_and_weight_gradient():
    x, w, a, b, dy, idx, s = make(333, 256, 384, 16, 3, 'cuda')
    with torch.no_grad():
        assert torch.equal(lora_linear(x, w, a, b, idx, 2.0), lora_linear(x, w, a, b, idx, torch.full((3,), 2.0, device='cuda')))
    # views: rows with a pitch, odd addresses
    wide = torch.zeros(333, 300, device='cuda', dtype=torch.bfloat16)
    wide[:, 3:259] = x
    with torch.no_grad():
        assert torch.equal(lora_linear(wide[:, 3:259], w, a, b, idx, s), lora_linear(x, w, a, b, idx, s))
        odd = torch.zeros(1 + w.numel(), device='cuda', dtype=torch.bfloat16)
        odd[1:] = w.flatten()
        assert torch.equal(lora_linear(x, odd[1:].view_as(w), a, b, idx, s), lora_linear(x, w, a, b, idx, s))
    clean = run_all((x, w, a, b, dy, idx, s))
    leaves = [t.clone().requires_grad_() for t in (w, a, b)]
    for t in leaves[1:]:
        t.main_grad = torch.ones_like(t, dtype=torch.float32)
    lora_linear(x, *leaves, idx, s).backward(dy)
    assert leaves[1].grad is None and leaves[2].grad is None
    refs, bounds = reference(x, w, a, b, dy, idx, s)
    check(leaves[1].main_grad - 1, refs[2], bounds[2] + U, 2 * U)
    check(leaves[2].main_grad - 1, refs[3], bounds[3] + U, 2 * U)
    check(leaves[0].grad, dy.double().t() @ x.double(), (dy.double().abs().t() @ x.double().abs()) * 333 * U)
    assert clean[0].isfinite().all()


@pytest.mark.gpu
def test_captured_and_replayed_with_other_indices():
    x, w, a, b, dy, idx, s = make(200, 512, 640, 16, 6, 'cuda')
    static = [x.clone().requires_grad_(), a.clone().requires_grad_(), b.clone().requires_grad_()]
    static_idx, static_dy = idx.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lora_linear(static[0], w, static[1], static[2], static_idx, s)
        grads = torch.autograd.grad(y, static, static_dy)
    for seed in (5, 6):
        other = make(200, 512, 640, 16, 6, 'cuda', 'runs' if seed == 5 else 'mixed', seed=seed)
        with torch.no_grad():
            static[0].copy_(other[0]), static[1].copy_(other[2]), static[2].copy_(other[3])
        static_idx.copy_(other[5]), static_dy.copy_(other[4])
        graph.replay()
        eager = run_all((other[0], w, other[2], other[3], other[4], other[5], s))
        for got, want in zip((y.detach(), *grads), eager):
            assert torch.equal(got, want)


@pytest.mark.gpu
def test_two_streams_at_once():
    args = [make(150 + 50 * i, 1024, 512, 16, 5, 'cuda', seed=i) for i in range(2)]
    want = [run_all(a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(5):
        got = []
        for stream, a in zip(streams, args):
            with torch.cuda.stream(stream):
                got.append(run_all(a))
        torch.cuda.synchronize()
        for g, v in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(g, v))


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    import deep_ep
    refused = pytest.raises((AssertionError, deep_ep.EPException))
    for k, n, rank in ((12, 16, 8), (16, 12, 8), (16, 16, 12), (16, 16, 136)):
        x, w, a, b, dy, idx, s = make(5, k, n, rank, 2, 'cuda')
        with refused:
            lora_linear(x, w, a, b, idx, s)
    x, w, a, b, dy, idx, s = make(5, 64, 64, 8, 2, 'cuda')
    for bad in (lambda: lora_linear(x, w.clone().requires_grad_(), a, b, idx, s), lambda: lora_linear(x, w, a, b, idx.cpu(), s),
                lambda: lora_linear(x.float(), w, a, b, idx, s), lambda: lora_linear(x, w[:, :32], a, b, idx, s), lambda: lora_linear(x, w, a, b[:1], idx, s),
                lambda: lora_linear(x, w, a, b[:, :32], idx, s), lambda: lora_linear(x, w, a, b, idx[:4], s), lambda: lora_linear(x, w, a, b, idx.float(), s),
                lambda: lora_linear(x, w, a, b, idx, s[:1]), lambda: lora_linear(x, w, a, b, idx, s.double()), lambda: lora_linear(x[0], w, a, b, idx, s),
                lambda: lora_linear(x, w, a[0], b, idx, s), lambda: lora_linear(x, w.cpu(), a, b, idx, s)):
        with refused:
            bad()


@pytest.mark.gpu
def test_second_derivatives_are_refused_where_they_are_taken():
    x, w, a, b, dy, idx, s = make(9, 64, 64, 8, 2, 'cuda')
    a.requires_grad_()
    y = lora_linear(x, w, a, b, idx, s)
    plain, = torch.autograd.grad(y, a, dy, retain_graph=True)
    kept, = torch.autograd.grad(y, a, dy, create_graph=True)
    assert torch.equal(plain, kept)
    with pytest.raises(RuntimeError, match='differentiable once'):
        kept.sum().backward()
