"""Each of attention's kernels on shapes that reach it, which the plan's own account of
its launches shows: split forwards of 128-row workgroups, gradients split over several tiles
of either axis, and both unsplit, on bands, ragged lengths, odd widths and addresses."""
import math
import re

import pytest

from cpde_amd import hip
from test_gpu_attention import Case

pytestmark = pytest.mark.gpu


def launches(device, c, left, right):
    """(forward kernel, its splits, gradient kernel, key splits, query splits)"""
    plan = hip.Attention(device, c.type, *c.shape, left=left, right=right)
    text = plan.info()
    plan.destroy()
    print(f'[case] {c.dtype} {c.shape} left={left} right={right}: {text}', flush=True)
    m = re.fullmatch(r'forward attention_(\w+) splits (\d+), gradient attention_(\w+) key splits (\d+) query splits (\d+)', text)
    return m[1], int(m[2]), m[3], int(m[4]), int(m[5])


def tried(device, c, left, right, ql=None, kl=None):
    for b in range(c.shape[0]):
        for names, lengths in (('q dout', ql), ('k v', kl)):
            for name in names.split() if lengths else ():
                t = getattr(c, name)
                t[b, max(lengths[b], 0):] = math.nan
    c.run(device, left, right, ql=ql, kl=kl)
    c.against(left, right, ql=ql, kl=kl)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('shape,left,right,ql,kl,order,offset', [
    ((2, 64, 4096, 4, 4, 128), -1, -1, None, None, 'bthd', 0),
    ((2, 64, 4096, 4, 2, 128), -1, 0, None, None, 'bhtd', 0),
    ((2, 64, 4096, 4, 2, 72), -1, 0, [64, 31], [4096, 1500], 'bthd', 0),
    ((2, 70, 3000, 4, 2, 33), -1, -1, None, None, 'bhtd', 1),
    ((2, 70, 3000, 4, 2, 33), -1, -1, [5, 70], [3000, 70], 'tbhd', 0),
    ((3, 64, 2500, 2, 2, 64), 1000, -1, [64, 0, 64], [2500, 2500, 0], 'bthd', 0),
])
def test_split_forward(device, dtype, shape, left, right, ql, kl, order, offset):
    c = Case(dtype, *shape, order=order, offset=offset)
    forward, splits, gradient, _, query_splits = launches(device, c, left, right)
    assert forward == 'forward_k' and splits > 1
    assert gradient == 'gradient_k' and query_splits > 1
    tried(device, c, left, right, ql, kl)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('shape,left,right,ql,kl,order,offset', [
    ((2, 200, 3000, 2, 1, 100), 40, -1, None, None, 'bthd', 0),
    ((2, 200, 3000, 2, 1, 100), -1, -1, [200, 77], [3000, 1111], 'bhtd', 0),
    ((2, 200, 3000, 2, 1, 100), -1, -1, None, None, 'tbhd', 1),
    ((2, 1000, 400, 4, 1, 128), -1, 0, None, None, 'bthd', 0),
    ((2, 1000, 400, 4, 1, 128), -1, 0, [300, 1000], [400, 129], 'bthd', 0),
    ((2, 2000, 500, 4, 2, 40), -1, -1, [2000, 700], [500, 260], 'bthd', 0),
    ((1, 2000, 300, 4, 2, 64), -1, -1, None, None, 'htbd', 3),
])
def test_gradient_split_over_the_queries(device, dtype, shape, left, right, ql, kl, order, offset):
    c = Case(dtype, *shape, order=order, offset=offset)
    _, _, gradient, key_splits, _ = launches(device, c, left, right)
    assert gradient == 'gradient_k' and key_splits > 1 and shape[2] > 256
    tried(device, c, left, right, ql, kl)


RAGGED = [300, 0, 1, 129, 128, 127, 300, 300, 17, 256, 257, 64, 65, 200, 299, 33]
RAGGED_KEYS = [400, 400, 400, 128, 129, 300, 0, 1, 64, 257, 256, 399, 65, 33, 127, 384]


@pytest.mark.parametrize('dtype,dim', [('f32', 32), ('f32', 64), ('f16', 32), ('f16', 64), ('f16', 96), ('f16', 128), ('bf16', 32),
                                       ('bf16', 64), ('bf16', 96), ('bf16', 128), ('f32', 40), ('f16', 33), ('bf16', 72)])
@pytest.mark.parametrize('left,right,ragged,order,offset', [
    (-1, 0, False, 'bthd', 0), (-1, -1, True, 'bthd', 0), (-1, 0, True, 'bhtd', 0), (150, -1, True, 'bthd', 0),
    (-1, 0, False, 'tbhd', 1)])
def test_128_rows(device, dtype, dim, left, right, ragged, order, offset):
    c = Case(dtype, 16, 300, 400, 8, 8, dim, order=order, offset=offset)
    forward, splits, gradient, key_splits, query_splits = launches(device, c, left, right)
    assert (forward, splits, gradient, key_splits, query_splits) == ('forward_k', 1, 'gradient_k', 1, 1)
    tried(device, c, left, right, RAGGED if ragged else None, RAGGED_KEYS if ragged else None)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('shape,right,forward,gradient', [
    ((2, 1, 65, 4, 4, 64), -1, 'step_k', None),
    ((2, 16, 90, 4, 2, 64), 0, 'rows_k', None),
    ((2, 260, 1500, 4, 2, 64), -1, None, 'few_gradient_k'),
])
def test_small_sets(device, dtype, shape, right, forward, gradient):
    c = Case(dtype, *shape)
    got = launches(device, c, -1, right)
    assert forward in (None, got[0]) and gradient in (None, got[2])
    tried(device, c, -1, right)


def test_refusals(device):
    with pytest.raises(hip.CpdeError, match='null argument'):
        hip.check(hip.load().cpde_attention_info(None, None, 0))
