"""Orthogonalised matrices, flat and tall, on sizes whose products run on tiles of 64, 128 and
256, split and not, with ends inside the tiles: one step against double on the GPU."""
import pytest

from layers import orthogonal_far, orthogonal_first
from sequences import UNIT
from test_gpu_orthogonal import forward, matrices

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('count,rows,columns', [
    (1, 2051, 8200), (1, 8200, 2051),    # A split on 128-wide tiles
    (3, 1030, 4100), (3, 4100, 1030),    # A and its square on 64-wide ones
    (2, 2500, 2600), (2, 2600, 2500),    # both on 128-wide ones
    (1, 3001, 5003), (1, 5003, 3001), (1, 9016, 9000)])  # the next X, and all three, on 256-wide ones
def test_first_step(device, dtype, count, rows, columns):
    print(f'[case] orthogonal {dtype} {count}x{rows}x{columns}, one step', flush=True)
    x = matrices(count, rows, columns, dtype)
    got = forward(device, x, dtype, 1).double()
    want, far = orthogonal_first(x, dtype)
    assert ((got - want).abs() <= far).all()
    assert float((got - want).norm() / want.norm()) < orthogonal_far(dtype, max(rows, columns)) / 4 + UNIT[dtype]
