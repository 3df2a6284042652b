"""Embedding lookups and the table's gradient through the C ABI against float64."""
import math

import pytest
import torch

from cpde_amd import hip
from sequences import E, TYPES, UNIT

pytestmark = pytest.mark.gpu


def ids_of(kind, tokens, rows, seed=3):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(tokens, generator=g, dtype=torch.float64)
    ids = (u * rows).long().clamp(max=rows - 1)
    if kind == 'skewed':
        ids = (u ** 6 * rows).long().clamp(max=rows - 1)
    elif kind == 'one':
        ids[:] = rows // 2
    elif kind == 'outside':
        ids[::3] = -1
        ids[1::3] = torch.where(u[1::3] < 0.5, rows, rows + (1 << 20))
    return ids


def gradient(device, dtype, tokens, rows, width, kind='uniform', index=torch.int32, accumulate=False, pad=0, offset=0,
             scale=1.5):
    torch_type, number = TYPES[dtype]
    ids = ids_of(kind, tokens, rows)
    g = torch.Generator('cuda').manual_seed(2)

    def matrix(n, kind_of):
        flat = torch.empty(n * (width + pad) + offset, device='cuda', dtype=kind_of)[offset:]
        return flat.view(n, width + pad)[:, :width]

    dout = matrix(tokens, torch_type).normal_(generator=g)
    dtable = matrix(rows, torch.float32).normal_(generator=g)
    before = dtable.cpu().double()
    plan = hip.Embedding(device, number, rows, width, tokens, index_bytes=8 if index == torch.int64 else 4)
    on = ids.to(index).cuda()
    torch.cuda.synchronize()
    views = hip.Rows(dout.data_ptr(), width + pad), hip.Rows(dtable.data_ptr(), width + pad)
    plan.backward(on, tokens, *views, scale, accumulate)
    device.synchronize()
    got = dtable.cpu()
    if not accumulate:
        plan.backward(on, tokens, *views, scale, accumulate)
        device.synchronize()
        assert torch.equal(dtable.cpu(), got)   # the same bits again
    plan.destroy()
    inside = (ids >= 0) & (ids < rows)
    at = torch.where(inside, ids, rows)
    x = dout.cpu().double() * float(torch.tensor(scale, dtype=torch.float32))

    def sums(v):
        return torch.zeros(rows + 1, width, dtype=torch.float64).index_add_(0, at, v)[:rows]

    want = sums(x) + (before if accumulate else 0)
    count = torch.zeros(rows + 1, dtype=torch.float64).index_add_(0, at, torch.ones(tokens, dtype=torch.float64))[:rows]
    # a sum's roundings, one an addition, then its product and its sum with what was there
    far = (count[:, None] + 3) * E * (sums(x.abs()) + (before.abs() if accumulate else 0))
    off = (got.double() - want).abs()
    assert (off <= far).all(), float((off / far.clamp(min=1e-300)).max())


@pytest.mark.parametrize('tokens', [257, 4095, 5000, 16384, 16385])
@pytest.mark.parametrize('rows,width', [(3, 9), (8, 8), (303, 12), (12, 203), (1500, 31), (66000, 5)])
@pytest.mark.parametrize('kind', ['uniform', 'skewed', 'one', 'outside'])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_gradient_narrow_and_odd_rows(device, dtype, kind, tokens, rows, width):
    """Rows narrower than a wave's loads, tables of few rows, widths off every alignment; common tokens."""
    print(f'[case] narrow gradient {dtype} {kind} tokens={tokens} rows={rows} width={width}', flush=True)
    gradient(device, dtype, tokens, rows, width, kind, index=torch.int64 if width % 2 else torch.int32,
             accumulate=rows == 12, pad=3 if rows == 303 else 0, offset=1 if rows == 1500 else 0)


@pytest.mark.parametrize('tokens', [0, 1, 63, 65, 1000, 4096, 4097, 10000, 70001])
@pytest.mark.parametrize('rows,width', [(1, 64), (2, 3), (63, 512), (1000, 130), (1025, 8), (70000, 16)])
def test_gradient_sizes(device, tokens, rows, width):
    if tokens * width > 20_000_000:
        pytest.skip('more than the host needs to sum')
    print(f'[case] gradient tokens={tokens} rows={rows} width={width}', flush=True)
    gradient(device, 'f32', tokens, rows, width)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('kind', ['uniform', 'skewed', 'one', 'outside'])
@pytest.mark.parametrize('tokens,rows,width', [(3000, 500, 96), (20000, 3000, 264), (9000, 100000, 8)])
def test_gradient_frequencies(device, dtype, kind, tokens, rows, width):
    """Common tokens (whole runs and runs of runs), one token alone, ids outside the table."""
    print(f'[case] gradient {dtype} {kind} tokens={tokens} rows={rows} width={width}', flush=True)
    gradient(device, dtype, tokens, rows, width, kind)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('pad,offset,width', [(8, 0, 64), (3, 0, 64), (0, 1, 64), (0, 0, 63), (5, 3, 1)])
def test_gradient_layouts(device, dtype, pad, offset, width):
    print(f'[case] gradient layout {dtype} pad={pad} offset={offset} width={width}', flush=True)
    gradient(device, dtype, 2000, 300, width, 'skewed', torch.int64, pad=pad, offset=offset)


def test_gradient_of_wide_ids(device):
    """A list for the passes in memory, ids of eight bytes, some outside the table."""
    gradient(device, 'f16', 9000, 5000, 40, 'outside', torch.int64)


@pytest.mark.parametrize('tokens', [900, 6000])
def test_gradient_adds(device, tokens):
    gradient(device, 'bf16', tokens, 2000, 72, 'skewed', accumulate=True)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
@pytest.mark.parametrize('tokens,rows,width,pad,offset', [(1, 1, 1, 0, 0), (700, 50, 64, 0, 0), (333, 1000, 100, 4, 0),
                                                           (50, 9, 2056, 0, 0), (129, 40, 64, 0, 1), (5000, 70, 24, 8, 0)])
def test_lookup(device, dtype, index, tokens, rows, width, pad, offset):
    print(f'[case] lookup {dtype} tokens={tokens} rows={rows} width={width} pad={pad} offset={offset}', flush=True)
    torch_type, number = TYPES[dtype]
    ids = ids_of('outside' if tokens > 1 else 'uniform', tokens, rows)
    if index == torch.int64 and tokens > 1:
        ids[0], ids[-1] = (1 << 32) + 1, -(1 << 40)  # (their low halves lie inside)
    flat = torch.empty(rows * (width + pad) + offset, device='cuda', dtype=torch_type)[offset:]
    table = flat.view(rows, width + pad)[:, :width].normal_(generator=torch.Generator('cuda').manual_seed(1))
    out = torch.full((tokens, width + pad), math.nan, device='cuda', dtype=torch_type)
    plan = hip.Embedding(device, number, rows, width, tokens, index_bytes=8 if index == torch.int64 else 4)
    on = ids.to(index).cuda()
    torch.cuda.synchronize()
    plan.forward(on, tokens, hip.Rows(table.data_ptr(), width + pad), hip.Rows(out.data_ptr(), width + pad), 3.7)
    device.synchronize()
    plan.destroy()
    inside = ((ids >= 0) & (ids < rows))[:, None]
    scale = float(torch.tensor(3.7, dtype=torch.float32))
    want = torch.where(inside, table.cpu().double()[ids.clamp(0, rows - 1)] * scale, 0.0)
    # one product in float and one rounding to the type
    off = (out[:, :width].cpu().double() - want).abs()
    assert (off <= (UNIT[dtype] + 2 * E) * want.abs() + 2.0 ** -25 * (dtype == 'f16')).all()
    assert out[:, width:].isnan().all()


def test_gradient_is_the_lookups(device):
    """sum(lookup(table) * dout) is linear in the table: its differences are its gradient's products."""
    rows, width, tokens, scale = 40, 32, 500, 2.0
    ids = ids_of('skewed', tokens, rows).int().cuda()
    g = torch.Generator('cuda').manual_seed(4)
    table, step = (torch.randn(rows, width, generator=g, device='cuda') for _ in range(2))
    dout = torch.randn(tokens, width, generator=g, device='cuda')
    out, dtable = torch.empty_like(dout), torch.empty_like(table)
    plan = hip.Embedding(device, hip.F32, rows, width, tokens)
    loss = []
    for sign in (1, -1):
        at = table + sign * step
        torch.cuda.synchronize()
        plan.forward(ids, tokens, hip.Rows.of(at), hip.Rows.of(out), scale)
        device.synchronize()
        loss.append(float((out.double() * dout.double()).sum()))
    plan.backward(ids, tokens, hip.Rows.of(dout), hip.Rows.of(dtable), scale)
    device.synchronize()
    plan.destroy()
    # (float roundings of 16,000 products of size one)
    assert abs((loss[0] - loss[1]) / 2 - float((dtable.double() * step.double()).sum())) < 16000 * 8 * E


def test_recorded(device):
    rows, width, tokens = 3000, 64, 9000
    ids = torch.zeros(tokens, dtype=torch.int32, device='cuda')
    dout = torch.empty(tokens, width, device='cuda').normal_(generator=torch.Generator('cuda').manual_seed(1))
    dtable = torch.empty(rows, width, device='cuda')
    plan = hip.Embedding(device, hip.F32, rows, width, tokens)
    torch.cuda.synchronize()
    plan.backward(ids, tokens, hip.Rows.of(dout), hip.Rows.of(dtable))
    device.synchronize()
    device.capture_begin()
    plan.backward(ids, tokens, hip.Rows.of(dout), hip.Rows.of(dtable))
    replay = device.capture_end()
    device.synchronize()
    for seed in range(3):
        ids.copy_(ids_of('skewed', tokens, rows, seed).int())
        torch.cuda.synchronize()
        replay.launch()
        device.synchronize()
        replayed = dtable.clone()
        plan.backward(ids, tokens, hip.Rows.of(dout), hip.Rows.of(dtable))
        device.synchronize()
        assert torch.equal(dtable, replayed)
    replay.destroy()
    plan.destroy()


def refused(match, call):
    with pytest.raises(hip.CpdeError, match=match) as err:
        call()
    assert err.value.code == hip.EINVAL


def test_refusals(device):
    make = lambda *a, **k: hip.Embedding(device, *a, **k)
    refused('element type', lambda: make(-1, 8, 8, 8))
    refused('table size', lambda: make(hip.F32, 0, 8, 8))
    refused('table size', lambda: make(hip.F32, 8, 0, 8))
    refused('table size', lambda: make(hip.F32, 8, 1 << 23, 8))
    refused('token count', lambda: make(hip.F32, 8, 8, -1))
    refused('4 or 8', lambda: make(hip.F32, 8, 8, 8, index_bytes=2))
    plan = make(hip.F32, 8, 8, 10)
    ids, table = torch.zeros(10, dtype=torch.int32, device='cuda'), torch.ones(10, 8, device='cuda')
    torch.cuda.synchronize()
    rows = hip.Rows.of(table)
    refused('more tokens', lambda: plan.forward(ids, 11, rows, rows))
    refused('more tokens', lambda: plan.backward(ids, -1, rows, rows))
    refused('null tensor', lambda: plan.forward(None, 10, rows, rows))
    refused('null tensor', lambda: plan.backward(ids, 10, hip.Rows(None, 8), rows))
    refused('null argument', lambda: plan.forward(ids, 10, None, rows))
    refused('overlap', lambda: plan.forward(ids, 10, rows, hip.Rows(table.data_ptr(), 7)))
    refused('overlap', lambda: plan.backward(ids, 10, rows, hip.Rows(table.data_ptr(), 0)))
    refused('negative stride', lambda: plan.forward(ids, 10, hip.Rows(table.data_ptr(), -8), rows))
    plan.destroy()
