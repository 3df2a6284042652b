"""Cosines and sines of far and of near positions, relative to themselves."""
import math

import pytest
import torch

from cpde_amd import hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dim,base', [(64, 10000.0), (48, 500000.0), (34, 100.0)])
def test_turns_of_one(device, interleaved, dim, base):
    """Pairs (1, 0) turn into (cos, sin), off by the sine's own four units (2^-23 of the value
    each), a rounding, and angles in double on both sides (eight roundings of the angle): also
    where a sine or a cosine is small, which an angle in float would leave off by 2^-24."""
    g = torch.Generator().manual_seed(3)
    at = torch.cat([torch.arange(3000), torch.randint(0, 1 << 21, (2000,), generator=g)])[None]
    tokens, half = at.shape[1], dim // 2
    q = torch.zeros(1, tokens, 1, dim, device='cuda')
    first = slice(0, None, 2) if interleaved else slice(0, half)
    second = slice(1, None, 2) if interleaved else slice(half, None)
    q[..., first] = 1
    for backward in (False, True):
        plan = hip.Rotation(device, hip.F32, 1, tokens, 1, 0, dim, interleaved=interleaved, base=base, norm=False)
        out, given = torch.full_like(q, math.nan), at.int().cuda()
        torch.cuda.synchronize()
        if backward:
            plan.backward(hip.Heads.of(q), None, hip.Heads.of(q), None, hip.Heads.of(out), None, positions=given)
        else:
            plan.forward(hip.Heads.of(q), None, hip.Heads.of(out), None, positions=given)
        device.synchronize()
        plan.destroy()
        angle = at[0].double()[:, None] * base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        for got, want in ((out[0, :, 0, first], torch.cos(angle)), (out[0, :, 0, second], torch.sin(angle) * (-1 if backward else 1))):
            far = 5 * 2.0 ** -23 * want.abs() + 16 * 2.0 ** -53 * angle + 1e-13
            off = (got.cpu().double() - want).abs()
            assert (off <= far).all(), float((off / far).max())
