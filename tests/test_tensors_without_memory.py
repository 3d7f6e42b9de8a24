"""Tensors that claim a GPU and have no memory there (fake ones, subclasses that wrap other tensors) are refused on the host, before
anything is launched: these tests need no GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import deep_ep
from deep_ep.ops.embedding import embedding_grad, embedding_lookup
from deep_ep.ops.grad_norm import clip_grad_norm_, grad_norm
from deep_ep.ops.lora import lora_linear


class Wrapper(torch.Tensor):
    @staticmethod
    def __new__(cls, *shape, dtype=torch.float32):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device='cuda')

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f'{func} was called')


def fake(*shape, dtype=torch.float32):
    with FakeTensorMode():
        return torch.empty(shape, dtype=dtype, device='cuda')


@pytest.mark.filterwarnings('ignore')
@pytest.mark.parametrize('make', [fake, Wrapper])
@pytest.mark.parametrize('wanted', [False, True], ids=['without gradients', 'with gradients'])
def test_refused(make, wanted):
    refused = pytest.raises(deep_ep.EPException, match='without memory')
    bf16 = torch.bfloat16
    table, ids, rows = make(8, 128), make(3, dtype=torch.int64), make(3, 128)
    with refused:
        embedding_lookup(table.requires_grad_(wanted), ids)
    with refused:
        embedding_grad(rows, ids, 8, out=make(8, 128))
    with refused:
        grad_norm([table])
    with refused:
        clip_grad_norm_([make(8, 8)], 1.0)
    with refused:
        lora_linear(make(4, 128, dtype=bf16), make(128, 128, dtype=bf16), make(2, 8, 128, dtype=bf16).requires_grad_(wanted),
                    make(2, 128, 8, dtype=bf16), make(4, dtype=torch.int32), make(2))
