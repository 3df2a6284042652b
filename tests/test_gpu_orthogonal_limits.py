"""Orthogonalised updates at the limits of what plans take: the widest and the highest matrices,
and NaN beside finite ones."""
import math

import pytest
import torch

from cpde_amd import hip
from layers import orthogonal_far, orthogonal_first
from sequences import E, TYPES, UNIT
from test_gpu_orthogonal import forward, matrices

pytestmark = pytest.mark.gpu
WIDEST = 1 << 20


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('rows,columns', [(40, WIDEST), (9, WIDEST - 31), (WIDEST, 40)])
def test_widest_matrices(device, dtype, rows, columns):
    """One step of the widest and of the highest there are, against double on the GPU."""
    print(f'[case] orthogonal {dtype} 1x{rows}x{columns}, one step', flush=True)
    x = matrices(1, rows, columns, dtype)
    got = forward(device, x, dtype, 1).double()
    want, far = orthogonal_first(x, dtype)
    assert ((got - want).abs() <= far).all()
    assert float((got - want).norm() / want.norm()) < orthogonal_far(dtype, WIDEST) / 4 + UNIT[dtype]


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
def test_update_of_the_widest(device, dtype):
    """A call that is taken moves the momentum once, and the weights with it."""
    print(f'[case] update {dtype} 1x24x{WIDEST}', flush=True)
    rate, factor = 0.5, 0.75
    plan = hip.Orthogonal(device, TYPES[dtype][1], 1, 24, WIDEST, 1)
    weight, gradient = (matrices(1, 24, WIDEST, dtype, seed=i) for i in (1, 3))
    momentum = matrices(1, 24, WIDEST, 'f32', seed=2)
    m, w, g = (t.double().clone() for t in (momentum, weight, gradient))
    torch.cuda.synchronize()
    plan.update(*(hip.Matrices.of(t) for t in (gradient, momentum, weight)), rate, factor, 0.0, False)
    device.synchronize()
    plan.destroy()
    # (two roundings of float: of the product's sum, or of the product and the sum)
    assert ((momentum.double() - (factor * m + g)).abs() <= 2 * E * (factor * m.abs() + g.abs())).all()
    o, far = orthogonal_first(momentum, dtype)
    want = w - rate * o
    assert ((weight.double() - want).abs() <= rate * far + (UNIT[dtype] + 4 * E) * (want.abs() + rate * far)).all()


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('rows,columns', [(150, 300), (300, 150), (131, 515), (130, 130)])
def test_not_a_number_stays_in_its_matrix(device, dtype, rows, columns):
    """Of a batch in launches of their own products."""
    x = matrices(3, rows, columns, dtype)
    want = forward(device, x, dtype, 3)
    for at, value in ((0, math.nan), (1, math.inf), (2, math.nan)):
        y = x.clone()
        y[at, rows - 1, columns - 1] = value
        got = forward(device, y, dtype, 3)
        for i in range(3):
            assert got[i].isnan().any() if i == at else torch.equal(got[i], want[i])
