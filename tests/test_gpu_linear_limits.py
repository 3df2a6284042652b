"""Products at the limits of what plans take, and 16-bit activations far out."""
import math

import pytest
import torch

from cpde_amd import hip
from sequences import TINY, TYPES, UNIT
from test_gpu_linear import forward, plan_of, refused, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('which', ['dx', 'forward'])
def test_a_refused_call_leaves_everything(device, which):
    """2^23 tiles of 64 x 64: neither part of a call runs where one of them cannot."""
    rows = 1 << 29
    print(f'[case] linear bf16 {rows}x1x1, {which}', flush=True)
    plan = hip.Linear(device, hip.BF16, rows, 1, 1)
    one = torch.ones(1, 1, device='cuda', dtype=torch.bfloat16)
    many = torch.full((rows, 1), 7.0, device='cuda', dtype=torch.bfloat16)
    dweight, dbias = torch.full_like(one, 3.0), torch.full_like(one[0], 5.0)
    same = hip.Rows(one.data_ptr(), 0)  # (every row the same value)
    torch.cuda.synchronize()
    if which == 'forward':
        refused('too many workgroups', lambda: plan.forward(rows, same, rows_of(one), rows_of(many)))
    else:
        refused('too many workgroups',
                lambda: plan.backward(rows, same, rows_of(one), same, dx=rows_of(many), dweight=rows_of(dweight),
                                      dbias=dbias.data_ptr(), accumulate=True))
    device.synchronize()
    assert float(dweight) == 3 and float(dbias) == 5 and bool((many == 7).all())
    if which == 'dx':
        # the others alone are taken: 2^29 ones, exact in 32 bits
        plan.backward(rows, same, None, same, dweight=rows_of(dweight), dbias=dbias.data_ptr())
        device.synchronize()
        assert float(dbias) == rows
    plan.destroy()


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
    z = z.double()
    integral, density = torch.special.ndtr(z), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    for got, want, size in ((y, z * integral, z.abs() * integral),
                            (dx, integral + z * density, integral + z.abs() * density)):
        far = r * size + UNIT[dtype] * (want.abs() + r * size) + TINY[dtype]
        off = (got.double() - want).abs() - far
        assert (off <= 0).all(), (float(z[off.argmax()]), float(got[off.argmax()]), float(want[off.argmax()]))
