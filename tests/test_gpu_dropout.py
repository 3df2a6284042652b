"""Dropout through the C ABI: the mask bit for bit that of the published generator,
values against float64."""
import math

import pytest
import torch

from cpde_amd import hip
from sequences import E, TYPES, UNIT, keep

pytestmark = pytest.mark.gpu


def matrix(rows, columns, dtype, pad=0, offset=0, seed=1):
    flat = torch.empty(rows * (columns + pad) + offset, device='cuda', dtype=TYPES[dtype][0])[offset:]
    return flat.view(rows, columns + pad)[:, :columns].normal_(generator=torch.Generator('cuda').manual_seed(seed))


def rows_of(t):
    return hip.Rows(t.data_ptr(), t.stride(0))


def dropped(device, dtype, x, probability, seed, offset=0, residual=None, y=None):
    y = torch.full_like(x, math.nan) if y is None else y
    torch.cuda.synchronize()
    device.dropout(TYPES[dtype][1], *x.shape, rows_of(x), rows_of(y), probability, seed, offset,
                   residual=None if residual is None else rows_of(residual))
    device.synchronize()
    return y


def against(y, x, dtype, probability, seed, offset=0, residual=None):
    mask = keep(*x.shape, probability, seed, offset)
    up = 2.0 ** 32 / (2.0 ** 32 - round(probability * 2 ** 32)) if probability < 1 else 0.0
    x = torch.where(mask, x.cpu().double() * up, 0.0) if probability < 1 else torch.zeros(x.shape, dtype=torch.float64)
    r = residual.cpu().double() if residual is not None else torch.zeros_like(x)
    # the factor's rounding, a product's, a sum's, and one to the type (f16's smallest values apart)
    far = UNIT[dtype] * (x + r).abs() + 3 * E * (x.abs() + r.abs()) + 2.0 ** -25 * (dtype == 'f16')
    got = y.cpu().double()
    assert ((got - (x + r)).abs() <= far).all()
    if residual is None:
        assert torch.equal(got != 0, (x != 0) & (got != 0)) and not got[~mask].any()


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('rows,columns,pad,offset', [
    (1, 1, 0, 0), (1, 7, 0, 0), (3, 5, 0, 0), (729, 128, 0, 0), (100, 64, 8, 0), (100, 64, 4, 0), (33, 250, 3, 0),
    (50, 64, 0, 1), (4097, 9, 0, 0), (2, 100003, 0, 0)])
def test_values(device, dtype, residual, rows, columns, pad, offset):
    print(f'[case] dropout {dtype} residual={residual} {rows}x{columns} pad={pad} offset={offset}', flush=True)
    x = matrix(rows, columns, dtype, pad, offset)
    r = matrix(rows, columns, dtype, 0, 0, seed=2) if residual else None
    y = dropped(device, dtype, x, 0.3, 1234567890123456789, 17, r)
    against(y, x, dtype, 0.3, 1234567890123456789, 17, r)


@pytest.mark.parametrize('probability', [0.0, 1e-10, 0.5, 0.999, 1.0])
def test_probabilities(device, probability):
    x = matrix(300, 64, 'f32')
    y = dropped(device, 'f32', x, probability, 5)
    against(y, x, 'f32', probability, 5)
    if probability == 0:
        assert torch.equal(y, x)
    r = matrix(300, 64, 'f32', seed=3)
    if probability == 1:
        assert torch.equal(dropped(device, 'f32', x, 1.0, 5, residual=r), r)


@pytest.mark.parametrize('offset', [0, (1 << 32) - 3, 1 << 40, (1 << 64) - 5])
def test_counters(device, offset):
    """Counters past 32 bits, and round the end of 64."""
    x = matrix(40, 72, 'bf16')
    against(dropped(device, 'bf16', x, 0.5, (1 << 64) - 1, offset), x, 'bf16', 0.5, (1 << 64) - 1, offset)


def test_layout_does_not_change_the_mask(device):
    """An element's word goes by its row and column alone."""
    x = matrix(60, 40, 'f32', pad=3)
    padded = dropped(device, 'f32', x, 0.4, 9)
    assert torch.equal(dropped(device, 'f32', x.contiguous(), 0.4, 9), padded.contiguous())


def test_in_place_and_gradient(device):
    """The output may be an input; the gradient is the call itself, which is linear:
    differences over any step are its products."""
    x, dy = matrix(100, 48, 'f32'), matrix(100, 48, 'f32', seed=8)
    y = dropped(device, 'f32', x, 0.2, 77)
    dx = dropped(device, 'f32', dy, 0.2, 77)
    step = matrix(100, 48, 'f32', seed=9)
    change = dropped(device, 'f32', x + step, 0.2, 77).double() - y.double()
    bound = 8 * E * 1.25 * float(((x.abs() + step.abs()) * dy.abs()).double().sum())
    assert abs(float((change * dy.double()).sum() - (dx.double() * step.double()).sum())) <= bound
    r = matrix(100, 48, 'f32', seed=10)
    both = dropped(device, 'f32', x, 0.2, 77, residual=r)
    same = x.clone()
    assert torch.equal(dropped(device, 'f32', same, 0.2, 77, y=same), y)
    onto = r.clone()
    assert torch.equal(dropped(device, 'f32', x, 0.2, 77, residual=onto, y=onto), both)


def test_nothing_of_a_dropped_element_is_left(device):
    x = matrix(64, 64, 'f16')
    mask = keep(64, 64, 0.5, 3).cuda()
    x[~mask] = math.nan
    y = dropped(device, 'f16', x, 0.5, 3)
    assert y.isfinite().all() and not y[~mask].any()
    x[~mask] = math.inf
    assert not dropped(device, 'f16', x, 0.5, 3)[~mask].any()


def test_broadcast_rows(device):
    """One row for all (a stride of zero), dropped differently in each."""
    x = matrix(1, 64, 'f32').expand(50, 64)
    y = torch.empty(50, 64, device='cuda')
    against(dropped(device, 'f32', x, 0.5, 3, y=y), x, 'f32', 0.5, 3)


def test_past_32_bits(device):
    """More than 2^32 elements: the last ones against their own counters."""
    rows, columns = (1 << 20) + 3, 4104
    x = torch.ones(rows, columns, device='cuda', dtype=torch.bfloat16)
    y = dropped(device, 'bf16', x, 0.5, 11)
    first = (rows - 4) * columns
    assert first > 1 << 32 and first % 4 == 0
    want = keep(4, columns, 0.5, 11, first // 4)
    assert torch.equal(y[-4:].cpu() != 0, want)
    assert torch.equal(y[:4].cpu() != 0, keep(4, columns, 0.5, 11))


def test_recorded(device):
    x, r = matrix(300, 64, 'bf16'), matrix(300, 64, 'bf16', seed=2)
    y = dropped(device, 'bf16', x, 0.3, 5, residual=r)
    device.capture_begin()
    device.dropout(hip.BF16, 300, 64, rows_of(x), rows_of(y), 0.3, 5, residual=rows_of(r))
    replay = device.capture_end()
    device.synchronize()
    for _ in range(3):
        x.mul_(0.5)
        torch.cuda.synchronize()
        replay.launch()
        device.synchronize()
        against(y, x, 'bf16', 0.3, 5, residual=r)
    replay.destroy()


def refused(match, call):
    with pytest.raises(hip.CpdeError, match=match) as err:
        call()
    assert err.value.code == hip.EINVAL


def test_refusals(device):
    x = matrix(8, 8, 'f32')
    r = rows_of(x)
    torch.cuda.synchronize()
    refused('element type', lambda: device.dropout(3, 8, 8, r, r, 0.5, 1))
    for p in (-0.1, 1.5, math.nan):
        refused('probability', lambda: device.dropout(hip.F32, 8, 8, r, r, p, 1))
    refused('matrix size', lambda: device.dropout(hip.F32, -1, 8, r, r, 0.5, 1))
    refused('matrix size', lambda: device.dropout(hip.F32, 1 << 40, 1 << 40, r, r, 0.5, 1))
    refused('null tensor', lambda: device.dropout(hip.F32, 8, 8, hip.Rows(None, 8), r, 0.5, 1))
    refused('null argument', lambda: device.dropout(hip.F32, 8, 8, None, r, 0.5, 1))
    refused('overlap', lambda: device.dropout(hip.F32, 8, 8, r, hip.Rows(x.data_ptr(), 7), 0.5, 1))
    refused('negative stride', lambda: device.dropout(hip.F32, 8, 8, hip.Rows(x.data_ptr(), -8), r, 0.5, 1))
    device.dropout(hip.F32, 0, 8, r, r, 0.5, 1)
    device.dropout(hip.F32, 8, 0, r, r, 0.5, 1)
