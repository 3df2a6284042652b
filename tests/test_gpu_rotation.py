"""Heads' norms and rotations, and their gradients, through the C ABI against float64."""
import math

import pytest
import torch

from cpde_amd import hip
from layers import rotation
from sequences import TYPES, check

pytestmark = pytest.mark.gpu


def tensor(shape, dtype, order=(0, 1, 2), pad=0, offset=0, seed=1, scale=1.0, fill=None):
    """[batch][token][head][dim] with the first three axes in memory in `order`."""
    *lead, dim = shape
    sizes = [lead[a] for a in order]
    flat = torch.empty(math.prod(sizes) * (dim + pad) + offset, device='cuda', dtype=TYPES[dtype][0])[offset:]
    if fill is None:
        flat.normal_(0, scale, generator=torch.Generator('cuda').manual_seed(seed))
    else:
        flat.fill_(fill)
    t = flat.view(*sizes, dim + pad)[..., :dim]
    return t.permute(*(order.index(a) for a in range(3)), 3)


def run(device, dtype, batch, tokens, heads, kv_heads, dim, rotated=None, interleaved=False, norm=True, weights=True,
        positions=None, order=(0, 1, 2), pad=0, offset=0, base=10000.0, eps=1e-6, in_place=False, backward=True):
    print(f'[case] rotation {dtype} {batch}x{tokens}x{heads}+{kv_heads}x{dim} {rotated} {interleaved} {norm} {order} {pad} {offset}',
          flush=True)
    rotated = dim if rotated is None else rotated
    plan = hip.Rotation(device, TYPES[dtype][1], batch, tokens, heads, kv_heads, dim, rotated, interleaved, base, eps, norm,
                        backward)
    t = {}
    for i, (n, h) in enumerate((('q', heads), ('k', kv_heads))):
        shape = (batch, tokens, h, dim)
        t[n] = tensor(shape, dtype, order, pad, offset, 1 + i, 2.0)
        t[f'd{n}_out'] = tensor(shape, dtype, order, pad, offset, 3 + i)
        t[n + '_out'], t['d' + n] = (tensor(shape, dtype, order, pad, offset, fill=math.nan) for _ in range(2))
        t[n + '_weight'] = 1 + tensor((1, 1, 1, dim), dtype, seed=5 + i, scale=0.3)[0, 0, 0] if weights else None
        t[f'd{n}_weight'] = torch.full((dim,), math.nan, device='cuda', dtype=TYPES[dtype][0])
    at = positions if positions is not None else torch.arange(tokens).expand(batch, tokens)
    given = None if positions is None else positions.to('cuda', torch.int32).contiguous()
    before = {n: t[n].clone() for n in ('q', 'k', 'dq_out', 'dk_out')}
    if in_place:
        t['q_out'], t['k_out'] = t['q'], t['k']
    view = {n: hip.Heads.of(v) if v is not None and v.dim() == 4 and v.numel() else None for n, v in t.items()}
    torch.cuda.synchronize()
    plan.forward(view['q'], view['k'], view['q_out'], view['k_out'], t['q_weight'], t['k_weight'], given)
    device.synchronize()
    out = {n: t[n + '_out'].clone() for n in ('q', 'k')}
    if backward:
        if in_place:
            t['q'].copy_(before['q'])
            t['k'].copy_(before['k'])
            view['dq'], view['dk'] = view['dq_out'], view['dk_out']
            t['dq'], t['dk'] = t['dq_out'], t['dk_out']
            torch.cuda.synchronize()
        plan.backward(view['q'], view['k'], view['dq_out'], view['dk_out'], view['dq'], view['dk'], t['q_weight'],
                      t['k_weight'], t['dq_weight'], t['dk_weight'], given)
        device.synchronize()
    plan.destroy()
    for n, h in (('q', heads), ('k', kv_heads)):
        if not h:
            continue
        w = None if t[n + '_weight'] is None else t[n + '_weight'].cpu()
        want = rotation(before[n].cpu(), w, at.cpu(), rotated, interleaved, base, eps, norm, dtype,
                        before[f'd{n}_out'].cpu() if backward else None)
        check(out[n], *want['out'], n + '_out')
        if backward:
            check(t['d' + n], *want['dx'], 'd' + n)
            check(t[f'd{n}_weight'], *want['dweight'], f'd{n}_weight')
    return out


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('batch,tokens,heads,kv_heads,dim,rotated', [
    (1, 1, 1, 1, 2, 2), (2, 5, 4, 2, 32, 32), (1, 33, 3, 1, 64, 32), (2, 9, 6, 2, 80, 80), (3, 7, 2, 2, 128, 128),
    (1, 12, 5, 1, 96, 48), (2, 3, 2, 1, 256, 256), (1, 6, 2, 1, 7, 4), (1, 4, 2, 2, 40, 20), (2, 5, 1, 1, 24, 0),
    (1, 8, 2, 1, 129, 62), (1, 700, 4, 4, 32, 32), (1, 5, 2, 1, 255, 254), (2, 5, 3, 3, 1, 0)])
def test_values_and_gradients(device, dtype, interleaved, batch, tokens, heads, kv_heads, dim, rotated):
    run(device, dtype, batch, tokens, heads, kv_heads, dim, rotated, interleaved)


@pytest.mark.parametrize('order', [(0, 1, 2), (0, 2, 1), (2, 1, 0), (1, 0, 2)])
@pytest.mark.parametrize('pad,offset', [(0, 0), (8, 0), (4, 0), (3, 0), (0, 1)])
def test_strides_and_alignment(device, order, pad, offset):
    for dtype in ('f32', 'bf16'):
        run(device, dtype, 2, 6, 4, 2, 48, 32, order=order, pad=pad, offset=offset)


@pytest.mark.parametrize('norm,weights', [(False, True), (False, False), (True, False)])
def test_without_norm_or_weights(device, norm, weights):
    run(device, 'f32', 2, 10, 4, 2, 64, norm=norm, weights=weights)
    run(device, 'bf16', 2, 10, 4, 2, 36, 18, norm=norm, weights=weights)


@pytest.mark.parametrize('heads,kv_heads', [(4, 0), (0, 3)])
def test_one_side_alone(device, heads, kv_heads):
    run(device, 'bf16', 2, 10, heads, kv_heads, 64)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_positions(device, dtype):
    """Places without a token, the first and the last positions there are, an entry without tokens."""
    g = torch.Generator().manual_seed(4)
    at = torch.randint(0, 1 << 20, (4, 20), generator=g)
    at[0, ::3] = -1
    at[1] = -7
    at[2, :4] = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 0])
    run(device, dtype, 4, 20, 4, 2, 64, positions=at)
    run(device, dtype, 4, 20, 4, 2, 64, positions=at, base=500000.0, interleaved=True)


def test_places_without_a_token_leave_nothing(device):
    """NaN and infinities there reach neither results nor the weights' gradients."""
    plan = hip.Rotation(device, hip.BF16, 2, 8, 4, 2, 64)
    at = torch.arange(8).repeat(2, 1)
    at[1, 5:] = -1
    at = at.cuda().int()
    q, k, dq_out, dk_out = (tensor((2, 8, h, 64), 'bf16', seed=i) for i, h in enumerate((4, 2, 4, 2)))
    for t, x in ((q, math.nan), (k, math.inf), (dq_out, math.inf), (dk_out, math.nan)):
        t[1, 5:] = x
    outs = [torch.full_like(t, 7.0) for t in (q, k, q, k)]
    dw = [torch.full((64,), math.nan, device='cuda', dtype=torch.bfloat16) for _ in range(2)]
    view = [hip.Heads.of(t) for t in (q, k, dq_out, dk_out, *outs)]
    torch.cuda.synchronize()
    plan.forward(view[0], view[1], view[4], view[5], positions=at)
    plan.backward(view[0], view[1], view[2], view[3], view[6], view[7], dq_weight=dw[0], dk_weight=dw[1], positions=at)
    device.synchronize()
    plan.destroy()
    for t in outs:
        assert t.isfinite().all() and not t[1, 5:].any() and t[1, :5].any()
    assert all(t.isfinite().all() for t in dw)


def test_rows_of_zeros_and_large_values(device):
    """A row of zeros is divided by the root of eps; squares of f16's largest values stay inside float."""
    for dtype, x in (('f32', 0.0), ('f16', 65504.0), ('bf16', 1e18)):
        plan = hip.Rotation(device, TYPES[dtype][1], 1, 3, 1, 0, 64, backward=False)
        q = torch.full((1, 3, 1, 64), x, device='cuda', dtype=TYPES[dtype][0])
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        plan.forward(hip.Heads.of(q), None, hip.Heads.of(out), None)
        device.synchronize()
        plan.destroy()
        want = rotation(q.cpu(), None, torch.arange(3)[None], 64, False, 10000.0, 1e-6, True, dtype)['out']
        check(out, *want, 'out')


def test_in_place(device):
    run(device, 'bf16', 2, 9, 4, 2, 64, in_place=True)
    run(device, 'f32', 2, 9, 4, 2, 50, 34, in_place=True)


def test_many_tokens(device):
    """More groups of lanes than the gradient's workgroups take at once."""
    run(device, 'bf16', 3, 3001, 4, 1, 32)


def test_past_32_bits(device):
    """Entries of a cache more than 2^32 bytes apart."""
    stride = (1 << 31) + 64
    cache = torch.empty(2 * stride, device='cuda', dtype=torch.bfloat16)
    k = cache.as_strided((2, 9, 2, 64), (stride, 128, 64, 1), 16)
    k.copy_(tensor((2, 9, 2, 64), 'bf16', seed=2))
    before = k.clone()
    plan = hip.Rotation(device, hip.BF16, 2, 9, 0, 2, 64, backward=False)
    torch.cuda.synchronize()
    plan.forward(None, hip.Heads.of(k), None, hip.Heads.of(k))
    device.synchronize()
    plan.destroy()
    check(k, *rotation(before.cpu(), None, torch.arange(9).expand(2, 9), 64, False, 10000.0, 1e-6, True, 'bf16')['out'], 'k_out')


@pytest.mark.parametrize('batch,tokens', [(0, 4), (3, 0)])
def test_no_tokens(device, batch, tokens):
    plan = hip.Rotation(device, hip.F32, batch, tokens, 2, 1, 16)
    t = torch.full((4, 4, 2, 16), 7.0, device='cuda')
    dw = torch.full((16,), 7.0, device='cuda')
    view = hip.Heads(t.data_ptr(), 128, 32, 16)
    torch.cuda.synchronize()
    plan.forward(view, view, view, view)
    plan.backward(view, view, view, view, view, view, dq_weight=dw.data_ptr())
    device.synchronize()
    assert (t == 7).all() and not dw.any()
    plan.destroy()


def test_into_a_cache(device):
    """Keys of single tokens turned into their places in a cache; nothing else of it changes."""
    cache = torch.full((3, 50, 2, 64), 7.0, device='cuda', dtype=torch.bfloat16)
    q, k = tensor((3, 1, 4, 64), 'bf16'), tensor((3, 1, 2, 64), 'bf16', seed=2)
    q_out = torch.empty_like(q)
    at = torch.full((3, 1), 17, dtype=torch.int32, device='cuda')
    plan = hip.Rotation(device, hip.BF16, 3, 1, 4, 2, 64, backward=False)
    torch.cuda.synchronize()
    plan.forward(hip.Heads.of(q), hip.Heads.of(k), hip.Heads.of(q_out), hip.Heads.of(cache[:, 17:18]), positions=at)
    device.synchronize()
    check(cache[:, 17:18], *rotation(k.cpu(), None, at.cpu(), 64, False, 10000.0, 1e-6, True, 'bf16')['out'], 'k_out')
    cache[:, 17] = 7
    assert (cache == 7).all()
    plan.destroy()


def test_gradient_is_that_of_differences(device):
    """Along a random direction of q and its weight, in float; see the bound at the products' test."""
    plan = hip.Rotation(device, hip.F32, 2, 9, 3, 0, 32, rotated=16)
    q, dy = tensor((2, 9, 3, 32), 'f32'), tensor((2, 9, 3, 32), 'f32', seed=2)
    w = 1 + tensor((1, 1, 1, 32), 'f32', seed=3, scale=0.3)[0, 0, 0]
    out, dq, dw = torch.empty_like(q), torch.empty_like(q), torch.empty_like(w)
    view = [hip.Heads.of(t) for t in (q, out, dy, dq)]
    plan.backward(view[0], None, view[2], None, view[3], None, w, dq_weight=dw)
    ways = tensor((2, 9, 3, 32), 'f32', seed=4), tensor((1, 1, 1, 32), 'f32', seed=5)[0, 0, 0]
    h, sums = 2.0 ** -7, []
    for s in (1, -1):
        at, weight = q + s * h * ways[0], w + s * h * ways[1]
        torch.cuda.synchronize()
        plan.forward(hip.Heads.of(at), None, view[1], None, weight)
        device.synchronize()
        sums.append(float((out.double() * dy).sum()))
    slope = float((dq.double() * ways[0]).sum() + (dw.double() * ways[1]).sum())
    size = math.sqrt(float((dq.double() ** 2).sum() + (dw.double() ** 2).sum()))
    assert abs((sums[0] - sums[1]) / (2 * h) - slope) < 0.02 * size
    plan.destroy()


def test_same_bits_and_recorded(device):
    plan = hip.Rotation(device, hip.BF16, 2, 500, 4, 2, 64)
    q, k, dq_out, dk_out = (tensor((2, 500, h, 64), 'bf16', seed=i) for i, h in enumerate((4, 2, 4, 2)))
    outs = [torch.empty_like(t) for t in (q, k, q, k)]
    dw = [torch.empty(64, device='cuda', dtype=torch.bfloat16) for _ in range(2)]
    view = [hip.Heads.of(t) for t in (q, k, dq_out, dk_out, *outs)]

    def calls():
        plan.forward(view[0], view[1], view[4], view[5])
        plan.backward(view[0], view[1], view[2], view[3], view[6], view[7], dq_weight=dw[0], dk_weight=dw[1])

    def go():
        torch.cuda.synchronize()
        calls()
        device.synchronize()
        return [t.clone() for t in (*outs, *dw)]

    first = go()
    assert all(torch.equal(a, b) for a, b in zip(first, go()))
    device.capture_begin()
    calls()
    replay = device.capture_end()
    device.synchronize()
    for _ in range(4):
        q.mul_(0.75)
        k.add_(0.25)
        want = go()
        for t in (*outs, *dw):
            t.fill_(math.nan)
        torch.cuda.synchronize()
        replay.launch()
        device.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (*outs, *dw)))
    replay.destroy()
    plan.destroy()


def refused(match, call):
    with pytest.raises(hip.CpdeError, match=match) as err:
        call()
    assert err.value.code == hip.EINVAL


def test_refusals(device):
    make = lambda *a, **k: hip.Rotation(device, hip.F32, *a, **k)  # noqa: E731
    refused('negative size', lambda: make(-1, 2, 2, 1, 16))
    refused('heads', lambda: make(1, 2, 0, 0, 16))
    refused('heads', lambda: make(1, 2, -1, 3, 16))
    refused('wide', lambda: make(1, 2, 2, 1, 257))
    refused('wide', lambda: make(1, 2, 2, 1, 0))
    refused('rotated', lambda: make(1, 2, 2, 1, 16, rotated=18))
    refused('rotated', lambda: make(1, 2, 2, 1, 16, rotated=7))
    refused('base', lambda: make(1, 2, 2, 1, 16, base=0.0))
    refused('base', lambda: make(1, 2, 2, 1, 16, base=math.nan))
    refused('eps', lambda: make(1, 2, 2, 1, 16, eps=-1.0))
    refused('too many', lambda: make(1 << 16, 1 << 16, 2, 1, 16))
    plan, flat = make(2, 3, 2, 1, 16), make(2, 3, 2, 1, 16, backward=False)
    t = torch.zeros(2, 3, 2, 16, device='cuda')
    v = hip.Heads(t.data_ptr(), 96, 32, 16)
    torch.cuda.synchronize()
    refused('null argument', lambda: plan.forward(v, None, v, v))
    refused('null tensor', lambda: plan.forward(hip.Heads(None, 96, 32, 16), v, v, v))
    refused('negative stride', lambda: plan.forward(hip.Heads(t.data_ptr(), 96, -32, 16), v, v, v))
    refused('overlap', lambda: plan.forward(v, v, hip.Heads(t.data_ptr(), 96, 16, 16), v))
    refused('overlap', lambda: plan.forward(v, v, hip.Heads(t.data_ptr(), 0, 32, 16), v))
    refused('without a backward', lambda: flat.backward(v, v, v, v, v, v))
    for p in (plan, flat):
        p.destroy()
