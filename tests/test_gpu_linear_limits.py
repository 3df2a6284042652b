"""Calls of products that have too many tiles for one launch."""
import pytest
import torch

from cpde_amd import hip
from test_gpu_linear import refused, rows_of

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
