"""Embedding lookup and its gradient against the formulas in 64 bits.

Tolerances. A lookup is one fp32 product (two for scaled 8-bit entries) and one rounding to the result's type: at most
eps / 2 + 3 * 2^-24 relative, plus half the smallest subnormal of the type. A gradient is an fp32 sum of n terms in some order
(at most n * 2^-24 of the sum of magnitudes), one product, and one rounding."""
import math

import pytest
import torch

from deep_ep.ops.embedding import embedding_grad, embedding_lookup

U32 = 2.0 ** -24
SUBNORMAL = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def make_ids(tokens, rows, kind, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    if kind == 'same':
        ids = torch.full((tokens,), rows - 1)
    elif kind == 'masked':
        ids = torch.full((tokens,), -1)
    elif kind == 'few':
        ids = torch.randint(0, min(rows, 5), (tokens,), generator=gen)
    else:
        ids = torch.randint(0, rows, (tokens,), generator=gen)
        if kind == 'outside':
            # negative, just behind the table, far behind it
            pick = torch.randint(0, 4, (tokens,), generator=gen)
            far = 2 ** 40 if dtype == torch.int64 else 2 ** 30
            ids = torch.where(pick == 0, -ids - 1, torch.where(pick == 1, ids + rows, torch.where(pick == 2, ids + far, ids)))
    return ids.to(dtype).to(device)


def lookup_reference(table, ids, scale, sf=None):
    valid = (ids >= 0) & (ids < table.size(0))
    out = torch.zeros(ids.numel(), table.size(1), dtype=torch.float64, device=table.device)
    at = ids.flatten()[valid.flatten()].long()
    rows = table.float()[at].double()
    if sf is not None:
        rows = rows * sf[at].double().repeat_interleave(128, dim=1)
    out[valid.flatten()] = rows * float(torch.tensor(scale, dtype=torch.float32))
    return out


def grad_reference(dy, ids, rows, scale):
    """(sums, magnitudes, terms per row) in 64 bits"""
    valid = (ids >= 0) & (ids < rows)
    at, d = ids[valid].long(), dy[valid].double()
    s = float(torch.tensor(scale, dtype=torch.float32))
    zeros = lambda: torch.zeros(rows, dy.size(1), dtype=torch.float64, device=dy.device)      # noqa: E731
    count = torch.bincount(at, minlength=rows).to(torch.float64).unsqueeze(1)
    return zeros().index_add_(0, at, d) * s, zeros().index_add_(0, at, d.abs()) * abs(s), count


def check_lookup(out, ref):
    t = out.dtype
    tol = ref.abs() * (torch.finfo(t).eps / 2 + 3 * U32) + SUBNORMAL[t] / 2
    assert ((out.double().view(ref.shape) - ref).abs() <= tol).all()


def check_grad(out, dy, ids, scale, before=None):
    ref, magnitude, count = grad_reference(dy, ids, out.size(0), scale)
    t = out.dtype
    if before is not None:
        ref = ref + before.double()
    tol = ref.abs() * (torch.finfo(t).eps / 2 + U32) + magnitude * (count + 3) * U32 + SUBNORMAL[t] / 2
    assert ((out.double() - ref).abs() <= tol).all()
    untouched = count.squeeze(1) == 0
    expected = torch.zeros_like(out[untouched]) if before is None else before[untouched]
    assert torch.equal(out[untouched], expected)


# ------------------------------------------------------------------------------------------------ CPU
def test_cpu_forms_agree_with_the_formulas():
    table = torch.randn(50, 24, dtype=torch.float32)
    ids = make_ids(40, 50, 'outside', torch.int64, 'cpu').view(4, 10)
    out = embedding_lookup(table, ids, 3.0)
    assert out.shape == (4, 10, 24)
    check_lookup(out, lookup_reference(table, ids, 3.0))
    dy = torch.randn(40, 24)
    check_grad(embedding_grad(dy, ids, 50, 0.5), dy, ids.flatten(), 0.5)
    acc = torch.randn(50, 24)
    before = acc.clone()
    check_grad(embedding_grad(dy, ids, 50, 0.5, out=acc, accumulate=True), dy, ids.flatten(), 0.5, before)


def test_cpu_gradient_reaches_the_table_or_its_main_grad():
    table = torch.randn(9, 4, dtype=torch.float64).float().requires_grad_()
    ids = torch.tensor([[1, 1, -1], [8, 20, 1]])
    dy = torch.randn(2, 3, 4)
    embedding_lookup(table, ids, 2.0).backward(dy)
    expected = torch.zeros(9, 4)
    expected[1] = 2 * (dy[0, 0] + dy[0, 1] + dy[1, 2])
    expected[8] = 2 * dy[1, 0]
    assert torch.allclose(table.grad, expected, rtol=4 * 2.0 ** -23, atol=1e-6)
    table.grad = None
    table.main_grad = torch.ones(9, 4)
    embedding_lookup(table, ids, 2.0).backward(dy)
    assert table.grad is None and torch.allclose(table.main_grad, expected + 1, rtol=4 * 2.0 ** -23, atol=1e-6)


def test_refusals():
    table, ids = torch.randn(8, 128), torch.tensor([0, 1])
    for bad in (lambda: embedding_lookup(table, ids.float()), lambda: embedding_lookup(table[0], ids),
                lambda: embedding_lookup(table.double(), ids), lambda: embedding_lookup(table, ids, table_sf=torch.ones(8, 1)),
                lambda: embedding_lookup(table.to(torch.float8_e4m3fn), ids),
                lambda: embedding_lookup(table.to(torch.float8_e4m3fn), ids, table_sf=torch.ones(8, 2)),
                lambda: embedding_grad(torch.randn(3, 128), ids, 8), lambda: embedding_grad(torch.randn(2, 128), ids, 8, accumulate=True),
                lambda: embedding_grad(torch.randn(2, 128), ids, 8, out=torch.empty(8, 64)),
                lambda: embedding_grad(torch.randn(2, 128).bfloat16(), ids, 8, out=torch.empty(8, 128).bfloat16(), accumulate=True),
                lambda: embedding_grad(torch.randn(2, 128), ids, 8, out=torch.empty(8, 128).half())):
        with pytest.raises((AssertionError, RuntimeError)):
            bad()


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize('tokens,hidden', [(0, 64), (1, 7168), (1, 1), (3, 1003), (257, 130), (5000, 1024), (1000, 7168)])
def test_lookup(dtype, tokens, hidden):
    rows = 1000
    table = torch.randn(rows, hidden, device='cuda').to(dtype)
    for kind, idt in (('outside', torch.int64), ('any', torch.int32)):
        ids = make_ids(tokens, rows, kind, idt, 'cuda')
        out = embedding_lookup(table, ids, math.sqrt(hidden))
        assert out.dtype == dtype and out.shape == (tokens, hidden)
        check_lookup(out, lookup_reference(table, ids, math.sqrt(hidden)))


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,hidden', [(1, 128), (77, 1024), (4000, 384)])
def test_lookup_of_8_bit_entries(tokens, hidden):
    rows = 500
    table = (torch.randn(rows, hidden, device='cuda') * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    sf = torch.rand(rows, hidden // 128, device='cuda')
    ids = make_ids(tokens, rows, 'outside', torch.int64, 'cuda')
    out = embedding_lookup(table, ids, 0.37, table_sf=sf)
    assert out.dtype == torch.bfloat16
    check_lookup(out, lookup_reference(table, ids, 0.37, sf))
    # entries and scales as views with a row pitch, the entries off every wide boundary
    wide = torch.zeros(rows, hidden + 3, dtype=torch.uint8, device='cuda')
    wide[:, 3:] = table.view(torch.uint8)
    sf_wide = torch.zeros(rows, hidden // 128 + 5, device='cuda')
    sf_wide[:, 2:2 + hidden // 128] = sf
    again = embedding_lookup(wide[:, 3:].view(torch.float8_e4m3fn), ids, 0.37, table_sf=sf_wide[:, 2:2 + hidden // 128])
    assert torch.equal(out, again)


@pytest.mark.gpu
@pytest.mark.parametrize('offset,pitch', [(0, 264), (1, 257), (2, 258), (8, 272)])
def test_strided_and_unaligned_tables(offset, pitch):
    storage = torch.randn(300 * pitch + 8, device='cuda').to(torch.bfloat16)
    table = storage[offset:].as_strided((300, 256), (pitch, 1))
    ids = make_ids(400, 300, 'any', torch.int64, 'cuda')
    assert torch.equal(embedding_lookup(table, ids, 2.5), embedding_lookup(table.contiguous(), ids, 2.5))
    dy = torch.randn(400 * pitch + 8, device='cuda').to(torch.bfloat16)[offset:].as_strided((400, 256), (pitch, 1))
    assert torch.equal(embedding_grad(dy, ids, 300, 2.5), embedding_grad(dy.contiguous(), ids, 300, 2.5))
    out = torch.full((300 * pitch + 8,), 7.0, device='cuda')
    view = out[offset:].as_strided((300, 256), (pitch, 1))
    embedding_grad(dy, ids, 300, 2.5, out=view)
    check_grad(view, dy, ids, 2.5)
    view.fill_(7.0)
    assert (out == 7.0).all()          # nothing between the rows was written


@pytest.mark.gpu
@pytest.mark.parametrize('kind', ['any', 'same', 'few', 'masked', 'outside'])
@pytest.mark.parametrize('tokens,rows,hidden', [(1, 1, 8), (31, 100, 1003), (33, 40, 130), (2049, 70000, 64), (8192, 300, 96),
                                                (8193, 1200, 256), (17000, 511, 64), (40000, 129280, 64),
                                                (70001, 300000, 24)])
def test_gradient(tokens, rows, hidden, kind):
    ids = make_ids(tokens, rows, kind, torch.int64, 'cuda', seed=tokens)
    for dtype, out_type in ((torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)):
        dy = torch.randn(tokens, hidden, device='cuda').to(dtype)
        out = torch.full((rows, hidden), float('nan'), device='cuda', dtype=out_type)
        embedding_grad(dy, ids, rows, 0.7, out=out)
        check_grad(out, dy, ids, 0.7)
        again = embedding_grad(dy, ids.to(torch.int32) if kind != 'outside' else ids, rows, 0.7, out=torch.empty_like(out))
        assert torch.equal(out, again)
        if out_type == torch.float32:
            before = torch.randn(rows, hidden, device='cuda')
            acc = before.clone()
            embedding_grad(dy, ids, rows, 0.7, out=acc, accumulate=True)
            check_grad(acc, dy, ids, 0.7, before)


@pytest.mark.gpu
def test_gradient_of_nothing():
    ids = torch.empty(0, dtype=torch.int64, device='cuda')
    assert (embedding_grad(torch.empty(0, 16, device='cuda'), ids, 5) == 0).all()
    acc = torch.ones(5, 16, device='cuda')
    embedding_grad(torch.empty(0, 16, device='cuda'), ids, 5, out=acc, accumulate=True)
    assert (acc == 1).all()
    assert embedding_grad(torch.ones(3, 16, device='cuda'), torch.zeros(3, dtype=torch.int64, device='cuda'), 0).shape == (0, 16)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    import deep_ep
    table, ids = torch.randn(8, 128, device='cuda'), torch.tensor([0, 1], device='cuda')
    flat = torch.randn(1000, device='cuda')
    for bad in (lambda: embedding_lookup(table, ids.float()), lambda: embedding_lookup(table[0], ids), lambda: embedding_lookup(table.double(), ids),
                lambda: embedding_lookup(table, ids, table_sf=torch.ones(8, 1, device='cuda')), lambda: embedding_lookup(table.to(torch.float8_e4m3fn), ids),
                lambda: embedding_lookup(table.to(torch.float8_e4m3fn), ids, table_sf=torch.ones(8, 2, device='cuda')),
                lambda: embedding_lookup(table, ids.cpu()), lambda: embedding_lookup(table.t(), ids),
                lambda: embedding_grad(torch.randn(3, 128, device='cuda'), ids, 8), lambda: embedding_grad(torch.randn(2, 128, device='cuda'), ids.cpu(), 8),
                lambda: embedding_grad(flat[:20].view(2, 10), ids, 8, out=flat[10:90].view(8, 10)),
                lambda: embedding_grad(flat[:20].view(2, 10), ids, 8, out=flat[100:].as_strided((8, 10), (5, 1))),
                lambda: embedding_grad(flat[:20].view(2, 10), ids, 8, out=flat[100:180].view(10, 8).t())):
        with pytest.raises((AssertionError, deep_ep.EPException)):
            bad()


@pytest.mark.gpu
def test_non_finite_rows_stay_where_they_are():
    table = torch.randn(20, 256, device='cuda')
    table[3], table[4, 5] = float('nan'), float('inf')
    ids = torch.tensor([3, -1, 4, 7], device='cuda')
    out = embedding_lookup(table, ids, 2.0)
    assert out[0].isnan().all() and (out[1] == 0).all() and out[2, 5] == float('inf') and out[3].isfinite().all()
    dy = torch.randn(4, 256, device='cuda')
    dy[0], dy[1] = float('nan'), float('nan')
    grad = embedding_grad(dy, ids, 20)
    bad = grad.isnan().any(dim=1)
    assert bad[3] and bad.sum() == 1          # the masked row's NaN goes nowhere


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    rows, hidden = 300001, 8192               # 2.46e9 elements
    table = torch.empty(rows, hidden, dtype=torch.bfloat16, device='cuda')
    ids = torch.tensor([rows - 1, 0, rows // 2, rows - 2], device='cuda')
    values = torch.randn(4, hidden, device='cuda').to(torch.bfloat16)
    table[ids] = values
    assert torch.equal(embedding_lookup(table, ids, 1.0), values)
    del table
    grad = embedding_grad(values, ids, rows)
    assert torch.equal(grad[ids], values)
    assert not grad[1:rows // 2].any() and not grad[rows // 2 + 1:rows - 2].any()


@pytest.mark.gpu
def test_autograd_main_grad_other_stream_and_graph():
    torch.manual_seed(0)
    table = torch.randn(5000, 320, device='cuda').to(torch.bfloat16).requires_grad_()
    ids = make_ids(3000, 5000, 'outside', torch.int64, 'cuda').view(30, 100)
    dy = torch.randn(30, 100, 320, device='cuda').to(torch.bfloat16)
    embedding_lookup(table, ids, 1.5).backward(dy)
    check_grad(table.grad, dy.view(-1, 320), ids.flatten(), 1.5)
    # expanded gradient (stride 0), as a sum gives it
    expanded, = torch.autograd.grad(embedding_lookup(table, ids, 1.5).sum(), table)
    check_grad(expanded, torch.ones_like(dy.view(-1, 320)), ids.flatten(), 1.5)
    expected = table.grad.clone()
    main = table.detach().clone().requires_grad_()
    main.main_grad = torch.zeros(5000, 320, device='cuda')
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        embedding_lookup(main, ids, 1.5).backward(dy)
    torch.cuda.current_stream().wait_stream(stream)
    assert main.grad is None
    check_grad(main.main_grad, dy.view(-1, 320), ids.flatten(), 1.5)

    flat = ids.flatten()
    static_ids, static_dy = flat.clone(), dy.view(-1, 320).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = embedding_lookup(table.detach(), static_ids, 1.5)
        grad = embedding_grad(static_dy, static_ids, 5000, 1.5)
    for seed in (1, 2):
        static_ids.copy_(make_ids(3000, 5000, 'few' if seed == 1 else 'any', torch.int64, 'cuda', seed))
        static_dy.normal_()
        graph.replay()
        check_lookup(out, lookup_reference(table.detach(), static_ids, 1.5))
        check_grad(grad, static_dy, static_ids, 1.5)
    static_ids.copy_(flat), static_dy.copy_(dy.view(-1, 320))
    graph.replay()
    assert torch.equal(grad, expected)


@pytest.mark.gpu
def test_gradient_of_a_changed_empty_or_computed_table():
    ids = torch.tensor([[1, 3], [1, -1]], device='cuda')
    table = torch.randn(5, 32, device='cuda').requires_grad_()
    out = embedding_lookup(table, ids, 2.0)
    with torch.no_grad():
        table.zero_()                               # the gradient does not depend on the values
    out.sum().backward()
    expected = torch.zeros(5, 32, device='cuda')
    expected[1], expected[3] = 4.0, 2.0
    assert torch.equal(table.grad, expected)
    assert (torch.autograd.grad(embedding_lookup(table, ids[:0]).sum(), table)[0] == 0).all()
    # a table that is itself computed, and second derivatives
    grad, = torch.autograd.grad(embedding_lookup(table * 3, ids, 2.0).sum(), table)
    assert torch.equal(grad, 3 * expected)
    kept, = torch.autograd.grad(embedding_lookup(table, ids, 2.0).sum(), table, create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        kept.sum().backward()
