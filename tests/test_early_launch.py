"""Kernels that may begin beside the work before them, read as text: none lets its successor begin before its own wait is over.
The successor is not always a kernel of the same operator, and waits for this one only."""
import glob
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WAIT, START = 'cudaGridDependencySynchronize', 'cudaTriggerProgrammaticLaunchCompletion'


def kernels():
    for path in sorted(glob.glob(os.path.join(ROOT, 'deep_ep', 'include', 'deep_ep', '**', '*.cuh'), recursive=True)):
        with open(path) as f:
            text = re.sub(r'//[^\n]*', '', f.read())
        for body in text.split('__global__')[1:]:
            body = body[:re.search(r'\n}', body).end()]
            if START in body:
                yield pytest.param(body, id=re.search(r'(\w+_kernel)\(', body).group(1))


@pytest.mark.parametrize('body', list(kernels()))
def test_the_next_kernel_begins_after_this_one_has_waited(body):
    assert WAIT in body and body.index(WAIT) < body.index(START)


@pytest.mark.gpu
@pytest.mark.parametrize('before', ['copy', 'zeros', 'other stream'])
def test_captured_behind_work_that_is_no_kernel(before):
    """The first kernel of an operator behind a copy, a fill and a join of two streams in a captured graph."""
    from deep_ep.ops.embedding import embedding_lookup
    from deep_ep.ops.grad_norm import grad_norm
    from deep_ep.ops.lora import lora_linear
    from test_lora import make
    x, w, a, b, dy, idx, s = make(50, 256, 128, 16, 3, 'cuda')
    table, ids = torch.randn(100, 64, device='cuda'), torch.arange(50, device='cuda')
    calls = {lambda: embedding_lookup(static['table'], ids): 'table', lambda: grad_norm([static['table']]): 'table',
             lambda: lora_linear(static['x'], w, a, b, idx, s): 'x'}
    fresh = {'table': table, 'x': x}
    static = {k: torch.full_like(v, 9.0) for k, v in fresh.items()}
    side = torch.cuda.Stream()
    for call, name in calls.items():
        static[name].fill_(9.0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            if before == 'copy':
                static[name].copy_(fresh[name])
            elif before == 'zeros':
                static[name].zero_()
            else:
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    static[name].copy_(fresh[name]).mul_(2)
                torch.cuda.current_stream().wait_stream(side)
            got = call()
        graph.replay()
        static[name].copy_(fresh[name] * {'copy': 1, 'zeros': 0, 'other stream': 2}[before])
        assert torch.equal(got, call())


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [3, 100, 700])
def test_with_fills_of_new_memory_between_the_kernels(rows):
    """Torch's deterministic mode fills every new tensor, so a kernel of its own stands between any two of an operator."""
    from deep_ep.ops.lora import lora_linear
    from test_lora import make
    x, w, a, b, dy, idx, s = make(rows, 256, 2048, 16, 3, 'cuda')
    leaves = [t.requires_grad_() for t in (x, a, b)]
    run = lambda: (lambda y: [y, *torch.autograd.grad(y, leaves, dy)])(lora_linear(x, w, a, b, idx, s))            # noqa: E731
    want = run()
    torch.use_deterministic_algorithms(True)
    try:
        got = run()
    finally:
        torch.use_deterministic_algorithms(False)
    assert all(torch.equal(g, v) for g, v in zip(got, want))
