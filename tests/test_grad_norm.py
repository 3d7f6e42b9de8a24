"""Global gradient norm and clipping against the formulas in 64 bits.

Tolerances. At most eight squares are added in fp32 (8 * 2^-24 of their sum, so 4 * 2^-24 of the norm), the rest in fp64, and the
norm is rounded once: 6 * 2^-24 leaves room for fp64. The factor adds a sum and a quotient (2 * 2^-24), the product one more, and
the result is rounded to its type: eps / 2 + 9 * 2^-24 relative, plus half the smallest subnormal."""
import math

import pytest
import torch
import torch.distributed as dist

from deep_ep.ops.grad_norm import clip_grad_norm_, grad_norm
from dist_utils import run_distributed

U32 = 2.0 ** -24
SUBNORMAL = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
SIZES = [1, 7, 0, 8, 129, 16384, 16385, 40000, 3]


def make(sizes, dtypes, device, scale=1.0, offset=0):
    """Tensors one after the other in one buffer per type, so that odd sizes leave odd alignments."""
    torch.manual_seed(len(sizes))
    flats = {t: (torch.randn(sum(sizes) + 8, device=device) * scale).to(t) for t in set(dtypes)}
    at, out = offset, []
    for i, n in enumerate(sizes):
        out.append(flats[dtypes[i % len(dtypes)]][at:at + n])
        at += n
    return out


def reference_norm(tensors):
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in tensors))


def check_norm(norm, tensors):
    ref = reference_norm(tensors)
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(float(norm) - ref) <= 6 * U32 * ref


def check_clipped(results, originals, max_norm):
    norm = reference_norm(originals)
    factor = min(1.0, max_norm / (norm + 1e-6))
    for r, o in zip(results, originals):
        ref = o.double() * factor
        tol = ref.abs() * (torch.finfo(r.dtype).eps / 2 + 9 * U32) + SUBNORMAL[r.dtype] / 2
        assert ((r.double() - ref).abs() <= tol).all()


MIXES = [[torch.bfloat16], [torch.float32], [torch.float16, torch.bfloat16, torch.float32]]
DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtypes', MIXES, ids=['bf16', 'fp32', 'mixed'])
@pytest.mark.parametrize('offset', [0, 1, 4])
def test_norm_and_clip(device, dtypes, offset):
    grads = make(SIZES, dtypes, device, offset=offset)
    before = [g.clone() for g in grads]
    check_norm(grad_norm(grads), before)
    # above the norm nothing changes, not by a bit
    check_norm(clip_grad_norm_(grads, 2 * reference_norm(before)), before)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    # into other tensors of other types, the gradients stay
    for out_type in (torch.bfloat16, torch.float32):
        out = make(SIZES, [out_type], device, offset=offset)
        check_norm(clip_grad_norm_(grads, 0.5, out=out), before)
        check_clipped(out, before, 0.5)
        assert all(torch.equal(g, b) for g, b in zip(grads, before))
    shifted = [torch.zeros(g.numel() + 3, dtype=g.dtype, device=device)[3:] for g in grads]      # another alignment than the gradient's
    clip_grad_norm_(grads, 0.5, out=shifted)
    check_clipped(shifted, before, 0.5)
    check_norm(clip_grad_norm_(grads, 0.5), before)
    check_clipped(grads, before, 0.5)


@pytest.mark.parametrize('device', DEVICES)
def test_zero_norm_limit_empty_lists_and_scalars(device):
    zero = [torch.zeros(100, device=device), torch.zeros((), device=device, dtype=torch.bfloat16)]
    assert float(clip_grad_norm_(zero, 1.0)) == 0 and not zero[0].any()
    assert float(grad_norm([])) == 0 and float(clip_grad_norm_([], 1.0)) == 0
    assert float(grad_norm([torch.empty(0, device=device)])) == 0
    g = torch.full((10,), 3.0, device=device)
    assert abs(float(grad_norm(t for t in (g, g[:5]))) - math.sqrt(135)) < 1e-5 and abs(float(grad_norm(g)) - math.sqrt(90)) < 1e-5
    assert abs(float(clip_grad_norm_(g, 0.0)) - math.sqrt(90)) < 1e-5 and not g.any()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('value', [1e25, 1e-30, 3e38], ids=str)
def test_values_whose_squares_leave_fp32(device, value):
    grads = [torch.full((1000,), value, device=device), torch.full((17,), value, device=device, dtype=torch.bfloat16)]
    ref = reference_norm(grads)
    norm = grad_norm(grads)
    if ref > 3.4e38:
        assert norm.isinf()
    else:
        assert abs(float(norm) - ref) <= 6 * U32 * ref


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('value', [float('nan'), float('inf')], ids=str)
def test_non_finite_gradients_show(device, value):
    grads = [torch.ones(5000, device=device), torch.ones(50, device=device, dtype=torch.bfloat16)]
    grads[0][4321] = value
    assert not grad_norm(grads).isfinite()
    norm = clip_grad_norm_(grads, 1.0)
    assert not norm.isfinite() and grads[0][4321].isnan()
    if math.isinf(value):
        assert float(norm) == value and not grads[1].any()
    else:
        assert norm.isnan() and grads[1].isnan().all()


@pytest.mark.parametrize('device', DEVICES)
def test_permuted_dense_tensors(device):
    base = torch.randn(6, 10, 4, device=device)
    t = base.permute(2, 0, 1)
    expected = base.clone()
    check_norm(clip_grad_norm_([t], 0.1), [expected])
    check_clipped([base], [expected], 0.1)


def test_refusals():
    g = torch.randn(10)
    for bad in (lambda: grad_norm([g.double()]), lambda: clip_grad_norm_([g], -1.0), lambda: clip_grad_norm_([g], 1.0, out=[]),
                lambda: clip_grad_norm_([g], 1.0, out=[torch.empty(9)]), lambda: grad_norm([g.long()])):
        with pytest.raises((AssertionError, RuntimeError)):
            bad()


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    import deep_ep
    g = torch.randn(100, device='cuda')
    before = g.clone()
    gaps = torch.randn(10, 10, device='cuda')[:, :5]
    for bad in (lambda: clip_grad_norm_([g, g], 1.0), lambda: clip_grad_norm_([g[:60], g[50:]], 1.0), lambda: grad_norm([gaps]),
                lambda: clip_grad_norm_([g[:50]], 1.0, out=[g[10:60]]), lambda: clip_grad_norm_([g.view(10, 10)], 1.0, out=[g.view(10, 10).t()]),
                lambda: clip_grad_norm_([g], 1.0, out=[g.view(torch.bfloat16)[:100]])):
        with pytest.raises((AssertionError, deep_ep.EPException)):
            bad()
    assert torch.equal(g, before)
    assert float(grad_norm([g, g])) > 0       # reading twice is fine


@pytest.mark.gpu
def test_many_tensors_and_repeatability():
    sizes = [(i * 977) % 4001 for i in range(2500)]
    grads = make(sizes, [torch.bfloat16, torch.float32], 'cuda')
    before = [g.clone() for g in grads]
    norms = [grad_norm(grads) for _ in range(3)]
    check_norm(norms[0], before)
    assert torch.equal(norms[0], norms[1]) and torch.equal(norms[0], norms[2])
    check_norm(clip_grad_norm_(grads, 1.0), before)
    check_clipped(grads, before, 1.0)


@pytest.mark.gpu
def test_more_than_2_to_32_bytes_in_one_tensor():
    g = torch.full((2 ** 31 + 17,), 0.5, device='cuda', dtype=torch.bfloat16)
    g[-1] = 4.0
    ref = math.sqrt((2 ** 31 + 16) * 0.25 + 16)
    assert abs(float(clip_grad_norm_([g], ref / 2)) - ref) <= 6 * U32 * ref
    assert float(g[-1]) == 2.0 and float(g[2 ** 31 + 15]) == 0.25 and float(g[0]) == 0.25


@pytest.mark.gpu
def test_captured_step_and_other_stream():
    grads = make([5000, 333, 70000], [torch.float32, torch.bfloat16], 'cuda')
    out = [torch.empty_like(g, dtype=torch.bfloat16) for g in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = clip_grad_norm_(grads, 1.0, out=out)
    for _ in range(2):
        for g in grads:
            g.normal_()
        graph.replay()
        check_norm(captured, grads)
        check_clipped(out, grads, 1.0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        norm = grad_norm(grads)
    torch.cuda.current_stream().wait_stream(stream)
    check_norm(norm, grads)


def _grouped_worker(rank, world):
    group = dist.group.WORLD
    torch.manual_seed(rank)
    mine = [torch.randn(50 + 10 * rank), torch.randn(7).bfloat16()]
    torch.manual_seed(99)
    shared = [torch.randn(30)]
    before = [t.clone() for t in mine + shared]
    norm = clip_grad_norm_(mine, 0.25, group=group, replicated=shared)
    gathered = [None] * world
    dist.all_gather_object(gathered, [t.double().square().sum().item() for t in before[:2]])
    ref = math.sqrt(sum(sum(g) for g in gathered) + before[2].double().square().sum().item())
    factor = 0.25 / (ref + 1e-6)
    ok = abs(float(norm) - ref) <= 6 * U32 * ref
    for t, b in zip(mine + shared, before):
        r = b.double() * factor
        ok = ok and bool(((t.double() - r).abs() <= r.abs() * (torch.finfo(t.dtype).eps / 2 + 9 * U32)).all())
    # a rank without gradients of its own takes part all the same
    alone = grad_norm([] if rank == 0 else [torch.ones(4)], group=group)
    assert ok and abs(float(alone) - 2.0 * math.sqrt(world - 1)) < 1e-6


def test_norm_over_ranks(master_port):
    run_distributed(_grouped_worker, 2, master_port)
