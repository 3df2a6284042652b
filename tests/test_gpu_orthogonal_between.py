"""Matrices that lie between one another's rows, and those that would overlap."""
import math

import pytest
import torch

from cpde_amd import hip
from sequences import TYPES
from test_gpu_orthogonal import forward, matrices, refused

pytestmark = pytest.mark.gpu


def interleaved(count, rows, columns, dtype, seed=None, pad=0):
    """[count][rows][columns] whose matrices take turns row by row in memory."""
    t = torch.full((rows, count, columns + pad), math.nan, device='cuda', dtype=TYPES[dtype][0])
    t = t.permute(1, 0, 2)[..., :columns]
    return t if seed is None else t.copy_(matrices(count, rows, columns, dtype, seed=seed))


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('count,rows,columns,pad', [(3, 20, 40, 0), (2, 150, 300, 5), (4, 1, 33, 0), (1, 150, 33, 2)])
def test_matrices_between_one_another(device, dtype, count, rows, columns, pad):
    print(f'[case] orthogonal {dtype} {count}x{rows}x{columns}, interleaved', flush=True)
    x = interleaved(count, rows, columns, dtype, 1, pad)
    want = forward(device, x.contiguous(), dtype, 2)
    out = interleaved(count, rows, columns, dtype, None, pad)
    assert torch.equal(forward(device, x, dtype, 2, out), want)
    plan = hip.Orthogonal(device, TYPES[dtype][1], count, rows, columns, 2)
    states = []
    for make in (interleaved, lambda *a: matrices(*a[:4], seed=a[4])):
        weight, momentum = make(count, rows, columns, dtype, 4), make(count, rows, columns, 'f32', 5)
        torch.cuda.synchronize()
        plan.update(*(hip.Matrices.of(t) for t in (x, momentum, weight)), 0.1)
        device.synchronize()
        states.append((weight, momentum))
    plan.destroy()
    assert all(torch.equal(a, b) for a, b in zip(*states))


def test_overlaps_are_refused(device):
    plan = hip.Orthogonal(device, hip.F32, 3, 5, 8)
    t = torch.zeros(3, 5, 8, device='cuda')
    v = hip.Matrices.of(t)
    torch.cuda.synchronize()
    for matrix, row in ((7, 24), (8, 23), (8, 16), (39, 8), (40, 7), (0, 8), (8, 0), (8, 8)):
        refused('overlap', lambda: plan.forward(v, hip.Matrices(t.data_ptr(), matrix, row)))
        refused('overlap', lambda: plan.update(v, hip.Matrices(t.data_ptr(), matrix, row), v, 0.1))
    plan.destroy()
