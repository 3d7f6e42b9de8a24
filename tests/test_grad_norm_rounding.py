"""The norm's error bound, from how its sums are made. The squares of 64 bytes (16 fp32 or 32 16-bit elements) are added in fp32
before they enter fp64 sums. A square goes through at most ten roundings on the way (eight in the chain of its 16 bytes, two where
four chains meet), so such a sum is off by at most 10 * 2^-24 of itself, the norm by half of that, 5 * 2^-24, and its own
rounding to fp32 adds 2^-24: 6 * 2^-24, and terms of second order and fp64's that 2^-40 covers. A clipped element adds the roundings of norm + 1e-6,
of the quotient and of the product, 3 * 2^-24, and the one to its type."""
import math

import pytest
import torch

from deep_ep.ops.grad_norm import clip_grad_norm_, grad_norm

U32 = 2.0 ** -24
DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize('count', [16, 32, 1000, 12345])
def test_norm_within_its_roundings(device, dtype, count):
    """Elements of one size (sums cross the same powers of two everywhere, so their errors have one sign) and of random sizes."""
    torch.manual_seed(count)
    values = [torch.full((count,), v, device=device).to(dtype) for v in torch.linspace(1.0, 2.0, 23).tolist()]
    values += [(torch.rand(count, device=device) + 0.5).to(dtype) for _ in range(8)]
    for g in values:
        ref = math.sqrt(math.fsum(g.double().square().tolist()))
        assert abs(float(grad_norm([g])) - ref) <= ref * (6 * U32 + 2.0 ** -40)
        out = torch.empty(count, device=device)
        clip_grad_norm_([g], 0.25, out=[out])
        want = g.double() * (0.25 / (ref + 1e-6))
        assert ((out.double() - want).abs() <= want.abs() * (10 * U32 + 2.0 ** -40)).all()
