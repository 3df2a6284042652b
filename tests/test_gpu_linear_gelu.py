"""GELU of 16-bit tensors far out, relative to its own values."""
import math

import pytest
import torch

from sequences import TINY, TYPES, UNIT
from test_gpu_linear import forward, plan_of, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', ['f16', 'bf16'])
def test_gelu_of_16_bits_keeps_its_digits(device, dtype):
    """Values and slopes far out on the left are as exact as the type there, relative to
    themselves: a formula for the normal integral off by r of its value r = 4e-5 at most (1e-6 of
    its own, exponents of up to 2^7 rounded to 2^-24 of themselves, twice: 2e-5, and float sums)."""
    r = 4e-5
    # (down to where the integral leaves float's normal range)
    z = torch.cat([torch.linspace(-12.5, 0, 3001), torch.linspace(0, 12.5, 500)]).to(TYPES[dtype][0]).cuda()[:, None]
    one = torch.ones(1, 1, device='cuda', dtype=z.dtype)
    plan = plan_of(device, dtype, len(z), 1, 1, 'gelu')
    y, pre = forward(device, plan, z, one, None, None)
    assert torch.equal(pre, z)
    dx = torch.full_like(z, math.nan)
    plan.backward(len(z), None, rows_of(one), rows_of(torch.ones_like(z)), pre=rows_of(z), dx=rows_of(dx))
    device.synchronize()
    plan.destroy()
    z, y, dx = (t.cpu().double() for t in (z, y, dx))
    integral, density = torch.erfc(-z / math.sqrt(2)) / 2, torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    for got, want, size in ((y, z * integral, z.abs() * integral),
                            (dx, integral + z * density, integral + z.abs() * density)):
        far = r * size + UNIT[dtype] * (want.abs() + r * size) + TINY[dtype]
        off = (got - want).abs() - far
        assert (off <= 0).all(), (float(z[off.argmax()]), float(got[off.argmax()]), float(want[off.argmax()]))
