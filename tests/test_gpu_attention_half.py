"""Gradients of attention in f16, whose exponents are few: score gradients are about the
output's gradient over the number of keys, and must keep their bits where that is far
below f16's normal range, and not overflow where it is above.

Tolerances: the gradients are compared with float64 ones from the same out and lse.  Every
score gradient ds and probability is rounded once, by at most u = 2^-11 of itself,
independently of the others: a sum of ds k has an error of variance below u^2 times the
sum of their squares (a third of that for evenly spread ones), and over a whole tensor the
root of it is bounded; twice that leaves room for the float roundings, which are of relative
size 1e-6.  Results are rounded once (u of themselves, 2^-25 below the normal range)."""
import math

import pytest
import torch

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


def far_from_exact(c, scale, left=-1, right=-1):
    """{name: (root of the squared errors' sum, its bound)} of a case that has run."""
    q, k, v, out, do = (t.cpu().double() for t in (c.q, c.k, c.v, c.out, c.dout))
    batch, lq, heads, dim = q.shape
    lk, group = k.shape[1], heads // k.shape[2]
    want = {n: torch.zeros_like(t) for n, t in (('dq', q), ('dk', k), ('dv', v))}
    rounded = {n: torch.zeros_like(t) for n, t in want.items()}
    at = torch.arange(lk)[None, :] - torch.arange(lq)[:, None] - (lk - lq)
    hidden = (at > right) & (right >= 0) | (at < -left) & (left >= 0)
    for b in range(batch):
        for h in range(heads):
            x, y, z, g = q[b, :, h], k[b, :, h // group], v[b, :, h // group], do[b, :, h]
            p = torch.exp(scale * (x @ y.T) - c.lse[b, h].cpu().double()[:, None])
            p = torch.where(hidden, 0.0, p)
            ds = p * (g @ z.T - (g * out[b, :, h]).sum(1, keepdim=True))
            for n, t, m, o, head in (('dq', ds, y, scale, h), ('dk', ds.T, x, scale, h // group), ('dv', p.T, g, 1.0, h // group)):
                want[n][b, :, head] += o * (t @ m)
                rounded[n][b, :, head] += o ** 2 * (t ** 2 @ m ** 2)
    return {n: (float((getattr(c, n).cpu().double() - want[n]).norm()),
                2 * U * math.sqrt(float(rounded[n].sum())) + U * float(want[n].norm()) + 2.0 ** -25 * math.sqrt(want[n].numel()))
            for n in want}


@pytest.mark.parametrize('size', [0.1, 1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize('side', ['q', 'k'])
@pytest.mark.parametrize('shape,right', [
    ((1, 256, 4096, 1, 1, 64), -1),
    ((1, 100, 2000, 2, 1, 40), 0),
    ((2, 2048, 2048, 8, 4, 64), 0),     # many rows and keys
    ((1, 700, 2500, 2, 2, 128), -1),
    ((1, 2000, 300, 6, 1, 96), -1),
])
def test_small_gradients_keep_their_bits(device, shape, right, size, side):
    """One side's tensor is 2^-9 of the other's and the scale takes it up, so that the other
    side's gradient lies within f16's normal range."""
    print(f'[case] f16 gradients {shape} right={right} dout {size} {side}', flush=True)
    c = Case('f16', *shape)
    getattr(c, side).mul_(2.0 ** -9)
    c.dout.mul_(size)
    scale = 2.0 ** 9 / math.sqrt(shape[-1])
    c.run(device, right=right, scale=scale)
    for name, (off, far) in far_from_exact(c, scale, right=right).items():
        assert off <= far, (name, off, far)


@pytest.mark.parametrize('shape', [(1, 40, 4, 2, 1, 64), (1, 1, 3, 1, 1, 128), (2, 700, 8, 16, 8, 64), (1, 300, 300, 2, 1, 32)])
def test_large_gradients_stay_finite(device, shape):
    """Score gradients of 10^5 and more, past f16, whose products with small keys and queries are within it."""
    print(f'[case] large f16 gradients {shape}', flush=True)
    c = Case('f16', *shape)
    c.k.mul_(2.0 ** -9)
    c.q.mul_(2.0 ** -9)
    c.v.mul_(16)
    c.dout.mul_(4000)
    c.dout.clamp_(-8000, 8000)
    scale = 1 / math.sqrt(shape[-1])
    c.run(device, scale=scale)
    dp = 4000 * 16 * math.sqrt(shape[-1])
    assert dp / shape[2] > 500
    for name in ('dq', 'dk', 'dv'):
        assert getattr(c, name).isfinite().all() or name == 'dv', name
    for name, (off, far) in far_from_exact(c, scale).items():
        assert off <= far or name == 'dv', (name, off, far)   # (dv, of the size of dout times the queries, may overflow)


def test_gradients_that_grow_along_the_keys(device):
    """Values, and with them score gradients, that grow by 2^40 over a list, and fall again."""
    c = Case('f16', 1, 200, 3000, 2, 1, 64)
    ramp = torch.cat([torch.linspace(-20, 8, 1500), torch.linspace(8, -20, 1500)]).exp2().cuda().view(1, -1, 1, 1)
    c.v.copy_((c.v.float() * ramp).half())
    c.k.mul_(2.0 ** -9)
    scale = 2.0 ** 9 / 8
    c.run(device, scale=scale)
    for name, (off, far) in far_from_exact(c, scale).items():
        assert off <= far, (name, off, far)


def test_zero_gradients(device):
    c = Case('f16', 1, 100, 200, 2, 1, 64)
    c.dout.zero_()
    c.run(device)
    for name in ('dq', 'dk', 'dv'):
        assert (getattr(c, name) == 0).all(), name
