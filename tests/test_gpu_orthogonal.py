"""Matrices brought near orthogonal ones, and the optimizer's step along them, through the
C ABI against float64."""
import math

import pytest
import torch

from cpde_amd import hip
from layers import orthogonal, orthogonal_far, orthogonal_first
from sequences import E, TYPES, UNIT, check

pytestmark = pytest.mark.gpu


def matrices(count, rows, columns, dtype, pad=0, offset=0, seed=1, scale=1.0, rank=None):
    flat = torch.empty(count * rows * (columns + pad) + offset, device='cuda', dtype=TYPES[dtype][0])[offset:]
    t = flat.view(count, rows, columns + pad)[..., :columns]
    g = torch.Generator('cuda').manual_seed(seed)
    if rank is None:
        t.normal_(0, scale, generator=g)
    else:
        a = torch.randn(count, rows, rank, device='cuda', generator=g)
        b = torch.randn(count, rank, columns, device='cuda', generator=g)
        t.copy_(torch.matmul(a, b) * scale)
    return t


def forward(device, x, dtype, steps, out=None):
    count, rows, columns = x.shape
    plan = hip.Orthogonal(device, TYPES[dtype][1], count, rows, columns, steps)
    out = torch.full((count, rows, columns), math.nan, device='cuda', dtype=x.dtype) if out is None else out
    torch.cuda.synchronize()
    plan.forward(hip.Matrices.of(x), hip.Matrices.of(out))
    device.synchronize()
    plan.destroy()
    return out


SIZES = [(1, 1, 1), (1, 1, 40), (3, 7, 5), (2, 16, 16), (1, 33, 70), (2, 64, 64), (1, 100, 257), (4, 128, 128), (1, 130, 129),
         (2, 300, 72), (1, 40, 600), (1, 260, 512),
         (2, 64, 256), (1, 65, 256), (3, 32, 512), (2, 500, 17), (1, 33, 512), (2, 200, 61), (1, 16, 513), (4, 8, 129), (1, 1, 1000), (2, 700, 1)]


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('count,rows,columns', SIZES)
def test_first_step(device, dtype, count, rows, columns):
    print(f'[case] orthogonal {dtype} {count}x{rows}x{columns}, one step', flush=True)
    x = matrices(count, rows, columns, dtype)
    check(forward(device, x, dtype, 1), *orthogonal_first(x.cpu(), dtype), 'out')


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('count,rows,columns', SIZES + [(1, 1000, 333), (2, 512, 768), (6, 24, 2000)])
def test_five_steps(device, dtype, count, rows, columns):
    print(f'[case] orthogonal {dtype} {count}x{rows}x{columns}', flush=True)
    x = matrices(count, rows, columns, dtype, scale=1e-3)
    got, want = forward(device, x, dtype, 5).double(), orthogonal(x, 5)
    for i in range(count):
        far = float((got[i] - want[i]).norm() / want[i].norm())
        assert far < orthogonal_far(dtype, max(rows, columns)), (i, far)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('rows,columns', [(1500, 2056), (2100, 1030), (9000, 9016)])
def test_large_matrices(device, dtype, rows, columns):
    """One step on tiles of every size, against double on the GPU."""
    print(f'[case] orthogonal {dtype} 1x{rows}x{columns}, one step', flush=True)
    x = matrices(1, rows, columns, dtype)
    got = forward(device, x, dtype, 1).double()
    want, far = orthogonal_first(x, dtype)
    assert ((got - want).abs() <= far).all()
    # and no further than roundings of both signs leave sums
    assert float((got - want).norm() / want.norm()) < orthogonal_far(dtype, columns) / 4 + UNIT[dtype]


@pytest.mark.parametrize('count,rows,columns', [(4, 15, 526), (1, 40, 700), (3, 8, 200), (2, 1100, 64), (1, 24, 480), (1, 1, 600),
                                                (1, 140, 2600)])
def test_even_singular_values(device, count, rows, columns):
    """Where A is nearly one number times the unit matrix, five steps of bf16 matrices are as
    exact as the type: what is rounded inside is off the diagonal only, a row of it at most
    0.3 of the diagonal (sqrt(rows / columns)), each to rms 2^-12 and weighed by 1.4 at most
    (4.775 of 3.44), independently in five steps whose errors later ones raise by 5 at most:
    under 0.3 * 1.4 * 2^-12 * sqrt(5) * 5 = 0.0011.  Rounding the result leaves 0.0017."""
    print(f'[case] orthogonal bf16 {count}x{rows}x{columns}, even', flush=True)
    x = matrices(count, rows, columns, 'bf16')
    got, want = forward(device, x, 'bf16', 5).double(), orthogonal(x, 5)
    least = float((want.bfloat16().double() - want).norm() / want.norm())
    far = float((got - want).norm() / want.norm())
    assert far < 1.25 * least, (far, least)


@pytest.mark.parametrize('count,rows,columns', [(2, 8, 32), (1, 16, 64), (4, 128, 128), (2, 60, 61)])
def test_small_float_matrices(device, count, rows, columns):
    """No further off than five steps of float products: those round A, b A + c A^2 and X to
    2^-24, where here diagonals and X itself are held so, and what is off the diagonal (a
    row of it about as large) to 2^-23 with two products in 2^-22 left out.  Over six matrices."""
    print(f'[case] orthogonal f32 {count}x{rows}x{columns}, small', flush=True)
    own = plain = 0.0
    for seed in range(6):
        x = matrices(count, rows, columns, 'f32', seed=seed)
        want = orthogonal(x, 5)
        y = (x.double() / x.double().square().sum((1, 2), keepdim=True).sqrt()).float()
        for _ in range(5):
            gram = y @ y.transpose(1, 2).contiguous()
            y = 3.4445 * y + (-4.7750 * gram + 2.0315 * (gram @ gram)) @ y
        own += float((forward(device, x, 'f32', 5).double() - want).norm())
        plain += float((y.double() - want).norm())
    assert own < 1.5 * plain, (own, plain)


def test_singular_values(device):
    """What it is for: singular vectors stay, values come into 0.68..1.13 (and the type's rounding)."""
    for dtype in ('f32', 'bf16'):
        x = matrices(1, 200, 300, dtype)
        got = forward(device, x, dtype, 5)[0].cpu().double()
        u, s, v = torch.linalg.svd(x[0].cpu().double(), full_matrices=False)
        inside = u.T @ got @ v.T
        assert 0.67 < float(inside.diag().min()) and float(inside.diag().max()) < 1.15
        assert float((inside - inside.diag().diag()).norm()) < orthogonal_far(dtype, 300) * float(got.norm()) + 1e-9


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_low_rank(device, dtype):
    """Directions without a share stay without one."""
    x = matrices(1, 96, 160, dtype, rank=3)
    if dtype == 'f32':
        # (a float matrix's roundings are a full-rank part of 6e-8 that the steps raise by 485)
        got, want = forward(device, x, dtype, 5).double(), orthogonal(x, 5)
        assert float((got - want).norm() / want.norm()) < 485 * orthogonal_far('f32', 160)
    else:
        got, want = forward(device, x, dtype, 2).double(), orthogonal(x, 2)
        assert float((got - want).norm() / want.norm()) < orthogonal_far('bf16', 160)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('pad,offset', [(0, 1), (3, 0), (8, 0), (5, 3)])
def test_strides_and_alignment(device, dtype, pad, offset):
    x = matrices(2, 50, 72, dtype, pad, offset)
    out = matrices(2, 50, 72, dtype, pad, offset)
    want = forward(device, x.contiguous(), dtype, 3)
    assert torch.equal(forward(device, x, dtype, 3, out), want)
    assert torch.equal(forward(device, x, dtype, 3, x), want)     # in place


def test_workspaces_start_with_anything(device):
    """Plans on memory that held NaN: what stands behind a width in them reaches no result."""
    held = [torch.full((size,), math.nan, device='cuda') for size in (1 << 16, 1 << 18, 1 << 20, 1 << 22) for _ in range(4)]
    torch.cuda.synchronize()
    del held
    torch.cuda.empty_cache()
    for dtype in ('f32', 'bf16'):
        for rows, columns in ((150, 33), (41, 300), (203, 515)):
            x = matrices(1, rows, columns, dtype)
            assert torch.equal(forward(device, x, dtype, 5), forward(device, x, dtype, 5))
            check(forward(device, x, dtype, 1), *orthogonal_first(x.cpu(), dtype), 'out')


def test_scale_and_zeros(device):
    """The size of a matrix does not count, from the type's smallest values to its largest; zeros give zeros."""
    x = matrices(1, 40, 56, 'f32')
    want = forward(device, x, 'f32', 5)
    for e in (-100, -30, 60, 120):
        assert torch.equal(forward(device, x * 2.0 ** e, 'f32', 5), want)
    x = torch.cat([torch.zeros_like(x), x])
    got = forward(device, x, 'f32', 5)
    assert not got[0].any() and torch.equal(got[1], want[0])
    x[0, 3, 4] = math.nan
    got = forward(device, x, 'f32', 5)
    assert got[0].isnan().any() and torch.equal(got[1], want[0])


def test_one_entry(device):
    """A single value is its sign times what the polynomial makes of one."""
    x = torch.zeros(2, 20, 30, device='cuda')
    x[0, 4, 7], x[1, 5, 6] = 1e-3, -5.0
    got = forward(device, x, 'f32', 5)
    s = 1.0
    for _ in range(5):
        s = 3.4445 * s - 4.775 * s ** 3 + 2.0315 * s ** 5
    assert abs(float(got[0, 4, 7]) - s) < 1e-5 and abs(float(got[1, 5, 6]) + s) < 1e-5
    got[0, 4, 7] = got[1, 5, 6] = 0
    assert not got.any()


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('nesterov', [False, True])
@pytest.mark.parametrize('count,rows,columns,pad', [(2, 64, 96, 0), (1, 130, 50, 3), (3, 9, 33, 0)])
def test_update(device, dtype, nesterov, count, rows, columns, pad):
    """Three steps in a row, each against float64 from the state before it."""
    print(f'[case] update {dtype} {count}x{rows}x{columns} nesterov={nesterov}', flush=True)
    rate, factor, decay = 0.05, 0.9, 0.1
    plan = hip.Orthogonal(device, TYPES[dtype][1], count, rows, columns)
    weight = matrices(count, rows, columns, dtype, pad, seed=1)
    momentum = matrices(count, rows, columns, 'f32', pad, seed=2)
    u = UNIT[dtype]
    for step in range(3):
        gradient = matrices(count, rows, columns, dtype, pad, seed=3 + step)
        m, w, g = (t.double().clone() for t in (momentum, weight, gradient))
        torch.cuda.synchronize()
        plan.update(hip.Matrices.of(gradient), hip.Matrices.of(momentum), hip.Matrices.of(weight), rate, factor, decay, nesterov)
        device.synchronize()
        m = factor * m + g
        check(momentum, m.cpu(), (3 * E * (m.abs() + factor * m.abs() + g.abs())).cpu(), 'momentum')
        o = orthogonal(g + factor * m if nesterov else m, 5)
        size = rate * math.sqrt(max(1, rows / columns))
        w = (1 - rate * decay) * w - size * o
        far = size * orthogonal_far(dtype, max(rows, columns)) * o.norm(dim=(1, 2), keepdim=True)
        off = (weight.double() - w).norm(dim=(1, 2), keepdim=True)
        assert (off <= far + (u + 8 * E) * w.norm(dim=(1, 2), keepdim=True)).all(), step
    plan.destroy()


def test_same_bits_and_recorded(device):
    plan = hip.Orthogonal(device, hip.BF16, 2, 96, 200)
    x, out = matrices(2, 96, 200, 'bf16'), torch.empty(2, 96, 200, device='cuda', dtype=torch.bfloat16)
    momentum, weight = matrices(2, 96, 200, 'f32', seed=4), matrices(2, 96, 200, 'bf16', seed=5)
    view = [hip.Matrices.of(t) for t in (x, out, momentum, weight)]

    def calls():
        plan.forward(view[0], view[1])
        plan.update(view[0], view[2], view[3], 0.02)

    kept = [t.clone() for t in (momentum, weight)]

    def go(launch):
        momentum.copy_(kept[0])
        weight.copy_(kept[1])
        out.fill_(math.nan)
        torch.cuda.synchronize()
        launch()
        device.synchronize()
        return [t.clone() for t in (out, momentum, weight)]

    first = go(calls)
    assert all(torch.equal(a, b) for a, b in zip(first, go(calls)))
    device.capture_begin()
    calls()
    replay = device.capture_end()
    device.synchronize()
    for _ in range(4):
        x.add_(0.25)
        assert all(torch.equal(a, b) for a, b in zip(go(calls), go(replay.launch)))
    replay.destroy()
    plan.destroy()


@pytest.mark.parametrize('count,rows,columns', [(0, 8, 8), (2, 0, 8), (2, 8, 0)])
def test_nothing(device, count, rows, columns):
    plan = hip.Orthogonal(device, hip.F32, count, rows, columns)
    plan.forward(hip.Matrices(None, 64, 8), hip.Matrices(None, 64, 8))
    plan.update(hip.Matrices(None, 64, 8), hip.Matrices(None, 64, 8), hip.Matrices(None, 64, 8), 0.1)
    plan.destroy()


def refused(match, call):
    with pytest.raises(hip.CpdeError, match=match) as err:
        call()
    assert err.value.code == hip.EINVAL


def test_refusals(device):
    make = lambda *a, **k: hip.Orthogonal(device, hip.F32, *a, **k)  # noqa: E731
    refused('negative size', lambda: make(-1, 8, 8))
    refused('too large', lambda: make(1, (1 << 20) + 1, 8))
    refused('too large', lambda: make(2000, 8, 8))
    refused('steps', lambda: make(1, 8, 8, steps=0))
    refused('steps', lambda: make(1, 8, 8, steps=100))
    plan = make(2, 8, 8)
    t = torch.zeros(2, 8, 8, device='cuda')
    v = hip.Matrices.of(t)
    torch.cuda.synchronize()
    refused('null argument', lambda: plan.forward(None, v))
    refused('null tensor', lambda: plan.forward(v, hip.Matrices(None, 64, 8)))
    refused('overlap', lambda: plan.forward(v, hip.Matrices(t.data_ptr(), 64, 7)))
    refused('overlap', lambda: plan.forward(v, hip.Matrices(t.data_ptr(), 63, 8)))
    refused('negative stride', lambda: plan.forward(hip.Matrices(t.data_ptr(), 64, -8), v))
    refused('finite', lambda: plan.update(v, v, v, math.nan))
    refused('finite', lambda: plan.update(v, v, v, 0.1, decay=math.inf))
    plan.destroy()
