"""Products with bias, activation and residual, and their gradients, through the C ABI
against float64."""
import math

import pytest
import torch

from cpde_amd import hip
from layers import ACTIVATIONS, linear, linear_gradient
from sequences import TYPES, check

pytestmark = pytest.mark.gpu


def matrix(rows, columns, dtype, pad=0, offset=0, seed=1, scale=1.0):
    flat = torch.empty(rows * (columns + pad) + offset, device='cuda', dtype=TYPES[dtype][0])[offset:]
    flat.normal_(0, scale, generator=torch.Generator('cuda').manual_seed(seed))
    return flat.view(rows, columns + pad)[:, :columns]


def rows_of(t):
    return hip.Rows(t.data_ptr(), t.stride(0))


def operands(dtype, rows, inputs, outputs, bias, residual, pad=0, offset=0):
    x = matrix(rows, inputs, dtype, pad, offset)
    w = matrix(outputs, inputs, dtype, pad, offset, 2, max(1, inputs) ** -0.5)
    b = matrix(1, outputs, dtype, 0, offset, 3)[0] if bias else None
    r = matrix(rows, outputs, dtype, pad, offset, 4) if residual else None
    return x, w, b, r


def plan_of(device, dtype, rows, inputs, outputs, kind, backward=True):
    return hip.Linear(device, TYPES[dtype][1], rows, inputs, outputs, ACTIVATIONS.index(kind), backward)


def forward(device, plan, x, w, b, r, pad=0, offset=0, pre=True, y=None):
    rows, outputs = x.shape[0], w.shape[0]
    y = torch.full((rows, outputs + pad), math.nan, device='cuda', dtype=x.dtype)[:, :outputs] if y is None else y
    z = torch.full((rows, outputs + pad), math.nan, device='cuda', dtype=x.dtype)[:, :outputs] if pre else None
    torch.cuda.synchronize()
    plan.forward(rows, rows_of(x), rows_of(w), rows_of(y), bias=None if b is None else b.data_ptr(),
                 residual=None if r is None else rows_of(r), pre=rows_of(z) if pre else None)
    device.synchronize()
    return y, z


SIZES = [  # rows, inputs, outputs: single ones, ends inside tiles, whole tiles, split sums, several tiles a side
    (1, 1, 1), (1, 64, 64), (2, 200, 72), (5, 7, 3), (16, 512, 256), (17, 2048, 40), (33, 64, 100), (64, 64, 64),
    (65, 72, 129), (128, 1024, 128), (130, 80, 260), (300, 33, 50), (257, 136, 257), (729, 128, 128), (48, 4096, 16)]


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('rows,inputs,outputs', SIZES)
def test_forward(device, dtype, rows, inputs, outputs):
    kind = ACTIVATIONS[(rows + inputs) % 5]
    print(f'[case] linear {dtype} {rows}x{inputs}x{outputs} {kind}', flush=True)
    x, w, b, r = operands(dtype, rows, inputs, outputs, True, outputs % 2 == 0)
    plan = plan_of(device, dtype, rows, inputs, outputs, kind)
    y, z = forward(device, plan, x, w, b, r)
    want = linear(x.cpu(), w.cpu(), b.cpu(), None if r is None else r.cpu(), kind, dtype)
    check(y, *want['y'], 'y')
    check(z, *want['pre'], 'pre')
    plan.destroy()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('pad,offset', [(0, 1), (1, 0), (4, 0), (8, 0), (3, 5)])
@pytest.mark.parametrize('rows,inputs,outputs', [(40, 96, 64), (200, 40, 136), (9, 130, 33)])
def test_strides_and_alignment(device, dtype, pad, offset, rows, inputs, outputs):
    print(f'[case] linear {dtype} {rows}x{inputs}x{outputs} pad={pad} offset={offset}', flush=True)
    x, w, b, r = operands(dtype, rows, inputs, outputs, True, True, pad, offset)
    plan = plan_of(device, dtype, rows, inputs, outputs, 'silu')
    y, z = forward(device, plan, x, w, b, r, pad)
    want = linear(x.cpu(), w.cpu(), b.cpu(), r.cpu(), 'silu', dtype)
    check(y, *want['y'], 'y')
    check(z, *want['pre'], 'pre')
    dy = matrix(rows, outputs, dtype, pad, offset, 5)
    gradient(device, plan, x, w, z, dy, 'silu', dtype, True)
    plan.destroy()


def gradient(device, plan, x, w, z, dy, kind, dtype, bias, accumulate=False, which=('dx', 'dweight', 'dbias')):
    torch.manual_seed(3)
    got = {'dx': torch.full(x.shape, math.nan, device='cuda', dtype=x.dtype),
           'dweight': torch.full(w.shape, math.nan, device='cuda', dtype=x.dtype),
           'dbias': torch.full((w.shape[0],), math.nan, device='cuda', dtype=x.dtype)}
    before = None
    if accumulate:
        for n in ('dweight', 'dbias'):
            got[n].normal_()
        before = {n: got[n].cpu().clone() for n in ('dweight', 'dbias')}
    torch.cuda.synchronize()
    plan.backward(x.shape[0], rows_of(x) if 'dweight' in which else None, rows_of(w) if 'dx' in which else None, rows_of(dy),
                  pre=rows_of(z) if kind != 'none' else None, dx=rows_of(got['dx']) if 'dx' in which else None,
                  dweight=rows_of(got['dweight']) if 'dweight' in which else None,
                  dbias=got['dbias'].data_ptr() if 'dbias' in which else None, accumulate=accumulate)
    device.synchronize()
    want = linear_gradient(x.cpu(), w.cpu(), None if z is None else z.cpu(), dy.cpu(), kind, dtype, before)
    for n in which:
        check(got[n], *want[n], n)
    for n in set(got) - set(which):
        assert got[n].isnan().all(), n
    return got


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('rows,inputs,outputs', SIZES)
def test_gradient(device, dtype, rows, inputs, outputs):
    kind = ACTIVATIONS[(rows + inputs + 2) % 5]
    print(f'[case] linear gradient {dtype} {rows}x{inputs}x{outputs} {kind}', flush=True)
    x, w, _, _ = operands(dtype, rows, inputs, outputs, False, False)
    z, dy = matrix(rows, outputs, dtype, seed=6, scale=2.0), matrix(rows, outputs, dtype, seed=7, scale=0.1)
    plan = plan_of(device, dtype, rows, inputs, outputs, kind)
    gradient(device, plan, x, w, z, dy, kind, dtype, True)
    gradient(device, plan, x, w, z, dy, kind, dtype, True, accumulate=True)
    plan.destroy()


@pytest.mark.parametrize('which', [('dx',), ('dweight',), ('dbias',), ('dx', 'dbias')])
@pytest.mark.parametrize('kind', ['none', 'gelu'])
def test_gradients_apart(device, which, kind):
    x, w, _, _ = operands('bf16', 70, 48, 40, False, False)
    z, dy = matrix(70, 40, 'bf16', seed=6), matrix(70, 40, 'bf16', seed=7)
    plan = plan_of(device, 'bf16', 70, 48, 40, kind)
    gradient(device, plan, x, w, z, dy, kind, 'bf16', True, which=which)
    plan.destroy()


@pytest.mark.parametrize('kind', ACTIVATIONS)
def test_activations_far_out(device, kind):
    """Values whose exponentials leave the range, infinities and NaN, through a product with one."""
    z = torch.tensor([0.0, -0.0, 1e-30, 5.0, -5.0, 20.0, -20.0, 88.0, -88.0, 104.0, -104.0, 1e4, -1e4, 3e38, -3e38, math.inf,
                      -math.inf, math.nan], device='cuda')[:, None]
    one = torch.ones(1, 1, device='cuda')
    plan = plan_of(device, 'f32', len(z), 1, 1, kind)
    y, pre = forward(device, plan, z, one, None, None)
    plan.destroy()
    z, y = z.double().cpu(), y.double().cpu()
    want = {'none': z, 'sigmoid': torch.sigmoid(z), 'relu': torch.relu(z), 'silu': z * torch.sigmoid(z),
            'gelu': z * torch.special.ndtr(z)}[kind]
    finite = want.isfinite()
    # (values of the definition 0 * infinity are NaN in both)
    assert torch.equal(finite, y.isfinite()) and torch.equal(want.isnan(), y.isnan())
    assert torch.equal(want[~finite & ~want.isnan()], y[~finite & ~want.isnan()])
    far = 16 * 2.0 ** -24 * (1 + z[finite].abs().clamp(max=200)) * want[finite].abs().clamp(max=200) + 2.0 ** -100
    near = want[finite].abs() <= 200
    assert ((y[finite] - want[finite]).abs()[near] <= far[near]).all()
    assert torch.equal(y[finite][~near], want[finite][~near])


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('rows,inputs,outputs', [(0, 8, 8), (8, 0, 8), (8, 8, 0), (0, 0, 0)])
def test_nothing_to_sum(device, dtype, rows, inputs, outputs):
    b = matrix(1, outputs, dtype)[0]
    x, w = (torch.zeros(s, device='cuda', dtype=TYPES[dtype][0]) for s in ((rows, inputs), (outputs, inputs)))
    plan = plan_of(device, dtype, 9, inputs, outputs, 'none')
    y = torch.full((9, max(1, outputs)), 7.0, device='cuda', dtype=x.dtype)
    dw, db = torch.full((max(1, outputs), max(1, inputs)), 7.0, device='cuda', dtype=x.dtype), torch.full_like(b, 7.0)
    torch.cuda.synchronize()
    dx = torch.full((9, max(1, inputs)), 7.0, device='cuda', dtype=x.dtype)
    view = {n: hip.Rows(t.data_ptr(), t.shape[1]) for n, t in (('x', x), ('w', w), ('y', y), ('dw', dw), ('dx', dx))}
    plan.forward(rows, view['x'], view['w'], view['y'], bias=b.data_ptr() if outputs else None)
    plan.backward(rows, view['x'], view['w'], view['y'], dx=view['dx'], dweight=view['dw'], dbias=db.data_ptr())
    device.synchronize()
    if outputs:
        assert torch.equal(y[:rows], b.expand(rows, outputs)) and (y[rows:] == 7).all()
    if rows == 0 and inputs and outputs:
        assert not dw.any() and not db.any()
    if outputs == 0 and inputs:
        assert not dx[:rows].any() and (dx[rows:] == 7).all()
    plan.destroy()


def test_rows_and_columns_behind_the_last_stay(device):
    """Results end where the matrices end."""
    x, w, b, _ = operands('bf16', 100, 64, 72, True, False)
    plan = plan_of(device, 'bf16', 128, 64, 72, 'relu')
    y = torch.full((110, 80), 7.0, device='cuda', dtype=torch.bfloat16)
    forward(device, plan, x, w, b, None, y=y[:100, :72])
    assert (y[100:] == 7).all() and (y[:, 72:] == 7).all()
    plan.destroy()


def test_what_stands_outside_is_not_read(device):
    """NaN beside the operands' columns and behind their rows."""
    for dtype in ('f32', 'bf16'):
        for inputs, outputs in ((72, 40), (70, 37)):
            big = torch.full((140, 88), math.nan, device='cuda', dtype=TYPES[dtype][0])
            wide = torch.full((60, 88), math.nan, device='cuda', dtype=TYPES[dtype][0])
            x, w = big[:130, :inputs], wide[:outputs, :inputs]
            x.normal_()
            w.normal_()
            plan = plan_of(device, dtype, 130, inputs, outputs, 'none')
            y, z = forward(device, plan, x, w, None, None)
            check(y, *linear(x.cpu(), w.cpu(), None, None, 'none', dtype)['y'], 'y')
            dy = torch.full((140, 88), math.nan, device='cuda', dtype=TYPES[dtype][0])[:130, :outputs]
            dy.normal_()
            gradient(device, plan, x, w, z, dy, 'none', dtype, True)
            plan.destroy()


def test_in_place_and_broadcast(device):
    """The residual may be the output; inputs may repeat one row."""
    x, w, b, r = operands('f32', 50, 40, 24, True, True)
    plan = plan_of(device, 'f32', 50, 40, 24, 'sigmoid')
    y, _ = forward(device, plan, x, w, b, r)
    same = r.clone()
    assert torch.equal(forward(device, plan, x, w, b, same, y=same)[0], y)
    one = x[:1].expand(50, 40)
    y, _ = forward(device, plan, one, w, b, r[:1].expand(50, 24))
    assert torch.equal(y, y[:1].expand(50, 24))
    plan.destroy()


def test_large_products(device):
    """Tiles of every size, float products on split operands, against double on the GPU."""
    for dtype, rows, inputs, outputs in (('bf16', 4096, 520, 4200), ('f16', 4100, 512, 4096), ('f32', 2100, 700, 1000),
                                         ('f32', 3000, 640, 1024)):
        print(f'[case] linear {dtype} {rows}x{inputs}x{outputs}', flush=True)
        x, w, b, r = operands(dtype, rows, inputs, outputs, True, True)
        plan = plan_of(device, dtype, rows, inputs, outputs, 'gelu')
        y, z = forward(device, plan, x, w, b, r)
        want = linear(x, w, b, r, 'gelu', dtype)
        for n, got in (('y', y), ('pre', z)):
            check(got, want[n][0].cpu(), want[n][1].cpu(), n)
        dy = matrix(rows, outputs, dtype, seed=5, scale=0.1)
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
        torch.cuda.synchronize()
        plan.backward(rows, rows_of(x), rows_of(w), rows_of(dy), pre=rows_of(z), dx=rows_of(dx), dweight=rows_of(dw),
                      dbias=db.data_ptr())
        device.synchronize()
        want = linear_gradient(x, w, z, dy, 'gelu', dtype)
        for n, got in (('dx', dx), ('dweight', dw), ('dbias', db)):
            check(got, want[n][0].cpu(), want[n][1].cpu(), n)
        # float results are as near as float sums of floats, not only within their worst case
        if dtype == 'f32':
            assert float((dx.double() - want['dx'][0]).norm() / want['dx'][0].norm()) < 2e-6
        plan.destroy()


@pytest.mark.parametrize('dtype,rows,inputs,outputs', [
    ('bf16', 300, 1001, 515), ('f16', 515, 520, 1030), ('f32', 203, 515, 333), ('f32', 1031, 264, 250), ('bf16', 3, 4100, 1003)])
@pytest.mark.parametrize('kind', ['none', 'silu'])
def test_odd_widths(device, dtype, rows, inputs, outputs, kind):
    """Widths that are not whole eights, over many tiles; a smaller call of the same plan."""
    print(f'[case] linear {dtype} {rows}x{inputs}x{outputs} {kind}', flush=True)
    x, w, b, r = operands(dtype, rows, inputs, outputs, True, True)
    plan = plan_of(device, dtype, rows, inputs, outputs, kind)
    dy = matrix(rows, outputs, dtype, seed=5, scale=0.1)
    for n in (rows, max(1, rows // 3)):
        y, z = forward(device, plan, x[:n], w, b, r[:n])
        want = linear(x[:n].cpu(), w.cpu(), b.cpu(), r[:n].cpu(), kind, dtype)
        check(y, *want['y'], 'y')
        check(z, *want['pre'], 'pre')
        gradient(device, plan, x[:n], w, z, dy[:n], kind, dtype, True)
    plan.destroy()


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('rows,inputs,outputs', [(33, 35, 41), (70, 9, 8), (66, 71, 65), (300, 129, 67), (3, 1031, 70), (129, 7, 200)])
def test_ends_of_odd_rows(device, dtype, rows, inputs, outputs):
    """Rows that end inside 16 bytes, NaN between them and around: none comes into a sum."""
    print(f'[case] linear {dtype} {rows}x{inputs}x{outputs} among NaN', flush=True)

    def among(rows, columns, seed):
        flat = torch.full((rows * (columns + 3) + 16,), math.nan, device='cuda', dtype=TYPES[dtype][0])
        t = flat[7:7 + rows * (columns + 3)].view(rows, columns + 3)[:, :columns]
        return t.copy_(matrix(rows, columns, dtype, seed=seed))

    x, w, dy = among(rows, inputs, 1), among(outputs, inputs, 2), among(rows, outputs, 5)
    for kind in ('none', 'silu'):
        plan = plan_of(device, dtype, rows, inputs, outputs, kind)
        y, z = forward(device, plan, x, w, None, None, pad=1)
        want = linear(x.cpu(), w.cpu(), None, None, kind, dtype)
        check(y, *want['y'], 'y')
        gradient(device, plan, x, w, z, dy, kind, dtype, True)
        plan.destroy()


@pytest.mark.parametrize('dtype', ['f16', 'bf16'])
@pytest.mark.parametrize('plan_rows,rows,inputs,outputs,kind,few', [
    (63, 63, 31, 61, 'gelu', 'both'), (400, 300, 40, 16, 'silu', 'both'), (16, 16, 2000, 24, 'relu', 'both'),
    (5000, 5000, 16, 32, 'sigmoid', 'both'), (20, 20, 100, 3000, 'gelu', 'dx'), (900, 900, 600, 100, 'silu', 'dweight'),
    (4000, 100, 600, 900, 'gelu', 'dx'), (64, 33, 257, 65, 'sigmoid', 'both')])
def test_few_gradients_are_rounded_once(device, dtype, plan_rows, rows, inputs, outputs, kind, few):
    """Gradients of few values are as far from those of `pre` as it stands as the exact ones
    rounded once: dz is a sum of two values (2^-17 of it left out, 2^-9 of half the result's rounding;
    f16: 2^-22), sums in 32 bits leave 2^-24 sqrt(5000) = 4e-6, slopes 16 * 2^-24 = 1e-6 where dz is of
    size one."""
    print(f'[case] linear gradient {dtype} {rows}x{inputs}x{outputs} {kind}, few', flush=True)
    x, w, b, _ = operands(dtype, rows, inputs, outputs, True, False)
    plan = plan_of(device, dtype, plan_rows, inputs, outputs, kind)
    _, z = forward(device, plan, x, w, b, None)
    dy = matrix(rows, outputs, dtype, seed=5)
    got = gradient(device, plan, x, w, z, dy, kind, dtype, True)
    want = linear_gradient(x, w, z, dy, kind, dtype)
    for n in ('dx', 'dweight'):
        if few in (n, 'both'):
            exact = want[n][0]
            least = float((exact.to(x.dtype).double() - exact).norm() / exact.norm())
            far = float((got[n].double() - exact).norm() / exact.norm())
            assert far < 1.01 * least + 1e-5, (n, far, least)
    again = gradient(device, plan, x, w, z, dy, kind, dtype, True, accumulate=True)
    assert torch.equal(again['dx'], got['dx'])
    plan.destroy()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_workspaces_start_with_anything(device, dtype):
    """Plans on memory that held NaN: what stands behind a width in them reaches no result."""
    held = [torch.full((size,), math.nan, device='cuda') for size in (1 << 10, 1 << 14, 1 << 18, 1 << 22) for _ in range(4)]
    torch.cuda.synchronize()
    del held
    torch.cuda.empty_cache()
    for rows, inputs, outputs in ((9, 130, 33), (70, 41, 77), (300, 515, 203)):
        x, w, b, r = operands(dtype, rows, inputs, outputs, True, True)
        plan = plan_of(device, dtype, rows, inputs, outputs, 'silu')
        y, z = forward(device, plan, x, w, b, r)
        check(y, *linear(x.cpu(), w.cpu(), b.cpu(), r.cpu(), 'silu', dtype)['y'], 'y')
        gradient(device, plan, x, w, z, matrix(rows, outputs, dtype, seed=5), 'silu', dtype, True)
        plan.destroy()


def test_gradient_is_that_of_differences(device):
    """Along a random direction of x, W and bias, in float: central differences of the sum of
    dy y.  With step h their truncation is h^2 / 6 of third derivatives (of order one a
    value), and float values' roundings are E sqrt(n) / h: both under 1e-3 of the slope."""
    rows, inputs, outputs = 64, 48, 40
    x, w, b, _ = operands('f32', rows, inputs, outputs, True, False)
    dy = matrix(rows, outputs, 'f32', seed=9)
    plan = plan_of(device, 'f32', rows, inputs, outputs, 'gelu')
    _, z = forward(device, plan, x, w, b, None)
    got = gradient(device, plan, x, w, z, dy, 'gelu', 'f32', True)
    g = torch.Generator('cuda').manual_seed(11)
    ways = [torch.randn(t.shape, device='cuda', generator=g) for t in (x, w, b)]
    h = 2.0 ** -7
    sums = [float((forward(device, plan, *(t + s * h * v for t, v in zip((x, w, b), ways)), None)[0].double() * dy).sum())
            for s in (1, -1)]
    slope = sum(float((got[n].double() * v).sum()) for n, v in zip(('dx', 'dweight', 'dbias'), ways))
    size = math.sqrt(sum(float((got[n].double() ** 2).sum()) for n in got))
    assert abs((sums[0] - sums[1]) / (2 * h) - slope) < 0.02 * size
    plan.destroy()


def test_same_bits_and_recorded(device):
    """The same call gives the same bits; recorded with its gradient, every replay too."""
    rows, inputs, outputs = 300, 1024, 136
    x, w, b, r = operands('bf16', rows, inputs, outputs, True, True)
    dy = matrix(rows, outputs, 'bf16', seed=5)
    plan = plan_of(device, 'bf16', rows, inputs, outputs, 'silu')
    y, z = torch.empty_like(r), torch.empty_like(r)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)

    def calls():
        plan.forward(rows, rows_of(x), rows_of(w), rows_of(y), bias=b.data_ptr(), residual=rows_of(r), pre=rows_of(z))
        plan.backward(rows, rows_of(x), rows_of(w), rows_of(dy), pre=rows_of(z), dx=rows_of(dx), dweight=rows_of(dw),
                      dbias=db.data_ptr())

    def run():
        torch.cuda.synchronize()
        calls()
        device.synchronize()
        return [t.clone() for t in (y, z, dx, dw, db)]

    first = run()
    assert all(torch.equal(a, c) for a, c in zip(first, run()))
    device.capture_begin()
    calls()
    replay = device.capture_end()
    device.synchronize()
    for _ in range(4):
        x.mul_(0.75)
        want = run()
        for t in (y, z, dx, dw, db):
            t.fill_(math.nan)
        torch.cuda.synchronize()
        replay.launch()
        device.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(want, (y, z, dx, dw, db)))
    replay.destroy()
    plan.destroy()


def test_callers_stream(device):
    """On a stream of the caller's, in order with its work and without a wait."""
    stream = torch.cuda.Stream()
    other = hip.Device(0, stream=stream.cuda_stream)
    x, w, b, r = operands('bf16', 256, 512, 128, True, True)
    plan = plan_of(device, 'bf16', 256, 512, 128, 'none')
    want, _ = forward(device, plan, x * 2, w, b, r)
    mine = plan_of(other, 'bf16', 256, 512, 128, 'none')
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        y = torch.empty_like(r)
        twice = x * 2
        mine.forward(256, rows_of(twice), rows_of(w), rows_of(y), bias=b.data_ptr(), residual=rows_of(r))
        got = y + 0
    stream.synchronize()
    assert torch.equal(got, want)
    for p in (plan, mine):
        p.destroy()
    other.close()


def test_past_32_bits(device):
    """Rows more than 2^32 bytes from the first, on both sides and in the gradients."""
    rows, inputs, outputs, stride = 70000, 64, 40, 32768
    big = torch.empty(rows * stride, device='cuda', dtype=torch.bfloat16).view(rows, stride)
    x, y, dy = big[:, :inputs], big[:, 128:128 + outputs], big[:, 256:256 + outputs]
    for t, seed in ((x, 1), (dy, 2)):
        t.copy_(matrix(rows, t.shape[1], 'bf16', seed=seed))
    w = matrix(outputs, inputs, 'bf16', seed=3, scale=0.125)
    plan = plan_of(device, 'bf16', rows, inputs, outputs, 'none')
    forward(device, plan, x, w, None, None, pre=False, y=y)
    last = slice(rows - 100, rows)
    check(y[last], *linear(x[last].cpu(), w.cpu(), None, None, 'none', 'bf16')['y'], 'y')
    dx, dw = torch.empty(rows, inputs, device='cuda', dtype=torch.bfloat16), torch.empty_like(w)
    torch.cuda.synchronize()
    plan.backward(rows, rows_of(x), rows_of(w), rows_of(dy), dx=rows_of(dx), dweight=rows_of(dw))
    device.synchronize()
    want = linear_gradient(x, w, None, dy, 'none', 'bf16')
    check(dx[last], *(t[last].cpu() for t in want['dx']), 'dx')
    check(dw, *(t.cpu() for t in want['dweight']), 'dweight')
    plan.destroy()


def refused(match, call):
    with pytest.raises(hip.CpdeError, match=match) as err:
        call()
    assert err.value.code == hip.EINVAL


def test_refusals(device):
    refused('element type', lambda: hip.check(hip.load().cpde_linear_create(device.handle, 7, 8, 8, 8, 0, 1,
                                                                            hip.ctypes.byref(hip.vp()))))
    refused('activation', lambda: hip.Linear(device, hip.F32, 8, 8, 8, 9))
    refused('negative size', lambda: hip.Linear(device, hip.F32, -1, 8, 8))
    refused('too large', lambda: hip.Linear(device, hip.F32, 8, 1 << 25, 8))
    x = torch.zeros(8, 8, device='cuda')
    r = rows_of(x)
    plan = hip.Linear(device, hip.F32, 8, 8, 8, hip.SILU)
    flat = hip.Linear(device, hip.F32, 8, 8, 8, hip.SILU, backward=False)
    torch.cuda.synchronize()
    refused('more rows', lambda: plan.forward(9, r, r, r))
    refused('more rows', lambda: plan.backward(-1, r, r, r, pre=r, dx=r))
    refused('null argument', lambda: plan.forward(8, None, r, r))
    refused('null tensor', lambda: plan.forward(8, r, hip.Rows(None, 8), r))
    refused('overlap', lambda: plan.forward(8, r, r, hip.Rows(x.data_ptr(), 7)))
    refused('stride', lambda: plan.forward(8, hip.Rows(x.data_ptr(), -8), r, r))
    refused('without a backward', lambda: flat.backward(8, r, r, r, pre=r, dx=r))
    refused('null argument', lambda: plan.backward(8, r, r, r, dx=r))                # pre of an activation
    refused('null argument', lambda: plan.backward(8, r, None, r, pre=r, dx=r))
    refused('null argument', lambda: plan.backward(8, None, r, r, pre=r, dweight=r))
    plan.backward(8, None, None, r, pre=r)                                           # nothing is asked for
    for p in (plan, flat):
        p.destroy()
