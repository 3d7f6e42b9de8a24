"""What `lora_linear` says that it takes as `scaling`, and takes."""
import typing

import pytest
import torch

from deep_ep.ops.lora import lora_linear
from test_lora import make

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


@pytest.mark.parametrize('device', DEVICES)
def test_a_number_or_a_tensor(device):
    assert typing.get_type_hints(lora_linear)['scaling'] == typing.Union[float, torch.Tensor]
    x, w, a, b, dy, idx, s = make(9, 64, 32, 8, 2, device)
    y = lora_linear(x, w, a, b, idx)
    assert torch.equal(y, lora_linear(x, w, a, b, idx, 1)) and torch.equal(y, lora_linear(x, w, a, b, idx, torch.ones(2, device=device)))
    with pytest.raises(TypeError):
        lora_linear(x, w, a, b, idx, None)
