"""Attention and its gradients through the C ABI against float64, within bounds
derived from the kernels' roundings (tests/sequences.py)."""
import math

import numpy as np
import pytest
import torch

from cpde_amd import hip
from sequences import TYPES, attention, check

pytestmark = pytest.mark.gpu


class Case:
    """Inputs, outputs (filled with NaN) and views of one shape."""

    def __init__(self, dtype, batch, queries, keys, heads, kv_heads, dim, seed=1, spread=1.0, offset=0, order='bthd',
                 shared=False):
        self.dtype, (torch_type, self.type) = dtype, TYPES[dtype]
        self.shape = (batch, queries, keys, heads, kv_heads, dim)
        g = torch.Generator('cuda').manual_seed(seed)

        def tensor(tokens, h, fill):
            # any order of the axes, `offset` elements into an allocation
            sizes = {'b': batch, 't': tokens, 'h': h, 'd': dim}
            flat = torch.empty(batch * tokens * h * dim + offset, device='cuda', dtype=torch_type)[offset:]
            t = flat.view([sizes[a] for a in order]).permute([order.index(a) for a in 'bthd'])
            return t.normal_(0, spread, generator=g) if fill else t.fill_(math.nan)

        self.q, self.k, self.v = tensor(queries, heads, True), tensor(keys, kv_heads, True), tensor(keys, kv_heads, True)
        if shared:  # one set of keys for the whole batch
            self.k, self.v = (t[:1].expand(batch, -1, -1, -1) for t in (self.k, self.v))
        self.dout = tensor(queries, heads, True)
        self.out, self.dq = tensor(queries, heads, False), tensor(queries, heads, False)
        self.dk, self.dv = tensor(keys, kv_heads, False), tensor(keys, kv_heads, False)
        self.lse = torch.full((batch, heads, queries), math.nan, device='cuda')
        torch.cuda.synchronize()

    def view(self, *names):
        return [hip.Heads.of(getattr(self, n)) for n in names]

    def run(self, device, left=-1, right=-1, scale=0.0, ql=None, kl=None, backward=True):
        plan = hip.Attention(device, self.type, *self.shape, scale=scale, left=left, right=right, backward=backward)
        lengths = [None if x is None else torch.tensor(x, dtype=torch.int32, device='cuda') for x in (ql, kl)]
        torch.cuda.synchronize()
        plan.forward(*self.view('q', 'k', 'v', 'out'), self.lse, *lengths)
        if backward:
            plan.backward(*self.view('q', 'k', 'v', 'out'), self.lse, *self.view('dout', 'dq', 'dk', 'dv'), *lengths)
        device.synchronize()
        plan.destroy()

    def against(self, left=-1, right=-1, scale=0.0, ql=None, kl=None, backward=True):
        want = attention(self.q, self.k, self.v, scale or self.shape[-1] ** -0.5, left, right, ql, kl,
                         self.dout if backward else None, self.dtype)
        for name, (value, far) in want.items():
            check(getattr(self, name), value, far, name)


SHAPES = [
    # (batch, queries, keys, heads, key heads, width)
    (1, 1, 1, 1, 1, 32),         # a single token
    (2, 1, 65, 4, 4, 16),        # one query row: the vector kernel, every lane width
    (3, 1, 130, 4, 2, 64),
    (2, 2, 300, 8, 2, 128),      # eight rows
    (1, 3, 40, 2, 1, 100),       # six
    (2, 33, 31, 3, 3, 32),       # matrix tiles from here
    (1, 129, 64, 2, 1, 64),
    (2, 70, 200, 5, 1, 96),      # five heads a key head
    (1, 150, 257, 3, 1, 128),
    (2, 64, 127, 4, 2, 80),
    (1, 9, 5, 1, 1, 40),
]


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('shape', SHAPES)
def test_shapes(device, dtype, shape):
    print(f'[case] attention {dtype} {shape}', flush=True)
    c = Case(dtype, *shape)
    c.run(device)
    c.against()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('queries,keys', [(100, 100), (100, 37), (37, 200), (1, 50), (4, 2), (140, 300)])
@pytest.mark.parametrize('left,right', [(-1, 0), (16, 0), (0, -1), (40, 7), (0, 0)])
def test_bands(device, dtype, queries, keys, left, right):
    """Causal and local bands, more queries than keys (rows that see nothing) and fewer."""
    print(f'[case] band {dtype} {queries} x {keys} left={left} right={right}', flush=True)
    c = Case(dtype, 2, queries, keys, 4, 2, 64)
    c.run(device, left, right)
    c.against(left, right)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('queries,keys,right', [(50, 90, -1), (50, 90, 0), (1, 400, -1), (2, 70, 0)])
def test_lengths(device, dtype, queries, keys, right):
    """Ragged batches: empty entries on either side, lengths out of range, and NaN and
    infinities past the lengths, which are not read."""
    print(f'[case] lengths {dtype} {queries} x {keys} right={right}', flush=True)
    c = Case(dtype, 6, queries, keys, 4, 2, 64)
    ql = [queries, 0, queries // 2 + 1, 1, queries + 5, -3]
    kl = [keys, keys, 0, 1, keys // 3, keys + 9]
    for b, (n, m) in enumerate(zip(ql, kl)):
        for t in (c.q, c.dout):
            t[b, max(n, 0):] = math.nan
        for t, x in ((c.k, math.inf), (c.v, math.nan)):
            t[b, max(m, 0):] = x
    c.run(device, right=right, ql=ql, kl=kl)
    c.against(right=right, ql=ql, kl=kl)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('right', [-1, 0])
@pytest.mark.parametrize('queries,keys', [(6, 700), (2, 4000)])
def test_lengths_of_few_rows(device, dtype, right, queries, keys):
    """Tiles of keys that every live row sees whole, and rows past the lengths beside them."""
    c = Case(dtype, 4, queries, keys, 6, 2, 64)
    ql, kl = [queries, queries // 2, 1, 0], [keys, keys - 100, 33, keys]
    c.run(device, right=right, ql=ql, kl=kl)
    c.against(right=right, ql=ql, kl=kl)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('order', ['bhtd', 'tbhd', 'htbd'])
@pytest.mark.parametrize('dim,offset', [(32, 0), (64, 3), (7, 0), (33, 1), (1, 0), (90, 0)])
def test_layouts(device, dtype, order, dim, offset):
    """Every order of the axes, addresses and widths that 16-byte accesses do not fit."""
    print(f'[case] layout {dtype} {order} dim={dim} offset={offset}', flush=True)
    c = Case(dtype, 2, 41, 70, 4, 2, dim, order=order, offset=offset)
    c.run(device, right=0)
    c.against(right=0)


def test_one_row_layouts(device):
    """The vector kernel on rows that 16-byte accesses do not fit."""
    for dim, offset, keys in ((7, 0, 30), (64, 1, 90), (128, 2, 700), (33, 0, 260)):
        print(f'[case] one row dim={dim} offset={offset}', flush=True)
        c = Case('f16', 2, 1, keys, 4, 2, dim, order='bhtd', offset=offset)
        c.run(device)
        c.against()


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('dim', [24, 64, 96, 128])
@pytest.mark.parametrize('left,right', [(-1, -1), (-1, 0), (50, 9)])
@pytest.mark.parametrize('queries,keys', [(330, 300), (300, 340)])
def test_workgroups_of_32_rows(device, dtype, dim, left, right, queries, keys):
    """Sets large enough for the kernels whose waves share out the other axis."""
    print(f'[case] 32 rows {dtype} {queries} x {keys} dim={dim} left={left} right={right}', flush=True)
    c = Case(dtype, 1, queries, keys, 4, 2, dim)
    c.run(device, left, right)
    c.against(left, right)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('order,dim,offset', [('bhtd', 40, 0), ('tbhd', 33, 0), ('bthd', 64, 1), ('htbd', 100, 0)])
def test_workgroups_of_32_rows_layouts(device, dtype, order, dim, offset):
    """The same on ragged batches (an empty entry on either side, NaN past the lengths) and other layouts."""
    print(f'[case] 32 rows {dtype} {order} dim={dim} offset={offset}', flush=True)
    c = Case(dtype, 4, 330, 340, 2, 1, dim, order=order, offset=offset)
    ql, kl = [330, 0, 201, 77], [340, 340, 0, 129]
    for b, (n, m) in enumerate(zip(ql, kl)):
        for t, x in ((c.q, n), (c.dout, n), (c.k, m), (c.v, m)):
            t[b, x:] = math.nan
    c.run(device, right=0, ql=ql, kl=kl)
    c.against(right=0, ql=ql, kl=kl)


@pytest.mark.parametrize('dtype,dim', [('f32', 32), ('f32', 64), ('f32', 96), ('f32', 128), ('f16', 32), ('f16', 64), ('f16', 96),
                                       ('f16', 128), ('bf16', 32), ('bf16', 64), ('bf16', 96), ('bf16', 128)])
def test_workgroups_of_128_rows(device, dtype, dim):
    """Many rows and keys: every workgroup resident more than once over."""
    c = Case(dtype, 4, 700, 900, 16, 8, dim)
    c.run(device, right=0)
    c.against(right=0)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('shape', [
    (1, 20, 3000, 2, 2, 64),     # few rows, many keys: forward and queries' gradients split
    (1, 3000, 20, 2, 1, 32),     # few keys, many rows: the keys' gradients split
    (1, 1, 5000, 2, 1, 128),     # one row over splits of the vector kernel
    (2, 1, 5000, 2, 2, 32),
    (1, 1, 3000, 2, 1, 50),
    (3, 2, 9000, 8, 2, 30),      # the same with lengths that leave splits empty, unaligned
])
def test_splits(device, dtype, shape):
    print(f'[case] splits {dtype} {shape}', flush=True)
    c = Case(dtype, *shape)
    kl = [shape[2], 5, shape[2] // 2][:shape[0]] if shape[0] > 1 else None
    c.run(device, kl=kl)
    c.against(kl=kl)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
def test_peaked_rows(device, dtype):
    """Scores of some hundreds (a row's weight on one key), whose maximum grows along the keys, and a scale."""
    c = Case(dtype, 1, 70, 300, 2, 1, 64, spread=4.0)
    c.k *= torch.linspace(0.1, 2, 300, device='cuda').view(1, -1, 1, 1).to(c.k.dtype)
    c.run(device, scale=0.5)
    c.against(scale=0.5)


def test_shared_keys(device):
    """Keys broadcast over the batch (a stride of zero): each entry's gradient is its own."""
    c = Case('f32', 4, 30, 50, 2, 2, 32, shared=True)
    c.run(device)
    c.against()
    c = Case('bf16', 3, 1, 50, 2, 1, 64, shared=True)
    c.run(device)
    c.against()


def test_infinities_in_keys(device):
    """A key whose score is -infinity has no weight; its value is finite."""
    c = Case('f32', 1, 40, 64, 1, 1, 32)
    c.q.abs_()
    c.k[0, 10] = -math.inf
    c.run(device, backward=False)
    keep = [j for j in range(64) if j != 10]
    want = attention(c.q, c.k[:, keep], c.v[:, keep], 32 ** -0.5)
    check(c.out, *want['out'], 'out')
    check(c.lse, *want['lse'], 'lse')


def test_no_keys_and_no_queries(device):
    c = Case('f32', 2, 3, 0, 2, 1, 32)
    c.run(device)
    assert (c.out == 0).all() and (c.lse == -math.inf).all() and (c.dq == 0).all()
    c = Case('bf16', 2, 0, 9, 2, 1, 32)
    c.run(device)
    assert (c.dk == 0).all() and (c.dv == 0).all()
    c = Case('bf16', 0, 5, 9, 2, 1, 32)
    c.run(device)


@pytest.mark.parametrize('token,keys', [
    (1 << 22, 540),     # a cache of 4.5 GB whose rows are read 16 bytes at a time
    (1 << 26, 40),      # rows further apart than a tile's 32-bit offsets reach
])
@pytest.mark.parametrize('queries', [1, 40])
def test_offsets_past_32_bits(device, token, keys, queries):
    c = Case('bf16', 1, queries, keys, 2, 1, 64)
    big = torch.empty(token * keys, dtype=torch.bfloat16, device='cuda')
    for name in 'kv':
        far = torch.as_strided(big, (1, keys, 1, 64), (0, token, 64, 1), 64 if name == 'v' else 0)
        far.copy_(getattr(c, name))
        setattr(c, name, far)
    torch.cuda.synchronize()
    c.run(device)
    c.against()


@pytest.mark.parametrize('shape', [(2, 200, 200, 4, 2, 64), (1, 20, 3000, 2, 2, 64), (1, 1, 5000, 2, 1, 128)])
def test_same_bits_again(device, shape):
    names = ('out', 'lse', 'dq', 'dk', 'dv')
    c = Case('bf16', *shape)
    c.run(device, right=0)
    first = [getattr(c, n).clone() for n in names]
    c.run(device, right=0)
    for n, f in zip(names, first):
        assert torch.equal(getattr(c, n), f), n


@pytest.mark.parametrize('which', ['q', 'k', 'v'])
def test_gradient_against_differences(device, which):
    """Central differences of sum(out * dout) along a random direction.  With h = 2^-7
    and tensors of size one the third-order term is under 1e-4 of |gradient| |direction|
    and the float sums' noise, 1e-6 / h of sqrt(elements), under 2e-4."""
    c = Case('f32', 1, 40, 60, 2, 1, 32)
    c.run(device, right=0)
    grad = getattr(c, 'd' + which).double()
    d = torch.randn(grad.shape, generator=torch.Generator('cuda').manual_seed(5), device='cuda')
    x, h, loss = getattr(c, which), 2.0 ** -7, []
    start = x.clone()
    for sign in (1, -1):
        x.copy_(start + sign * h * d)
        torch.cuda.synchronize()
        c.run(device, right=0, backward=False)
        loss.append(float((c.out.double() * c.dout.double()).sum()))
    slope = (loss[0] - loss[1]) / (2 * h)
    assert abs(slope - float((grad * d).sum())) < 1e-3 * float(grad.norm() * d.norm())


@pytest.mark.parametrize('shape', [(2, 1, 40, 2, 1, 64), (1, 20, 3000, 2, 2, 64), (2, 60, 70, 2, 1, 64), (4, 700, 900, 16, 8, 64)])
def test_statistics_are_optional(device, shape):
    """Inference asks for none; the outputs are the same bits."""
    c = Case('bf16', *shape)
    c.run(device, backward=False)
    out = c.out.clone()
    c.out.fill_(math.nan)
    c.lse = None
    c.run(device, backward=False)
    assert torch.equal(c.out, out)


def test_traced(device):
    """Tracing counts the operators' launches in classes of their own."""
    device.trace(True)
    c = Case('bf16', 1, 50, 60, 2, 1, 64)
    c.run(device)
    report = device.trace_report()
    device.trace(False)
    assert report['attention'][0] == 1 and report['attention_gradient'][0] == 1
    assert report['attention'][2] == 4 * 2 * 50 * 60 * 64
    c.against()


def test_callers_stream():
    """A device on a stream of torch's: ordered with torch's work there without a wait."""
    stream = torch.cuda.Stream()
    device = hip.Device(0, stream=stream.cuda_stream)
    c = Case('bf16', 4, 300, 300, 4, 4, 64)
    plan = hip.Attention(device, c.type, *c.shape)
    views = c.view('q', 'k', 'v', 'out')
    with torch.cuda.stream(stream):
        c.q.mul_(0.5)
        plan.forward(*views, c.lse)
        doubled = c.out * 2
    stream.synchronize()
    c.against(backward=False)
    assert torch.equal(doubled, c.out * 2)
    plan.destroy()
    device.close()


def test_recorded(device):
    """A recorded forward and backward replays on the buffers' present contents."""
    c = Case('bf16', 2, 100, 130, 4, 2, 64)
    plan = hip.Attention(device, c.type, *c.shape)

    def step():
        plan.forward(*c.view('q', 'k', 'v', 'out'), c.lse)
        plan.backward(*c.view('q', 'k', 'v', 'out'), c.lse, *c.view('dout', 'dq', 'dk', 'dv'))

    step()
    device.synchronize()
    device.capture_begin()
    step()
    replay = device.capture_end()
    device.synchronize()
    for _ in range(3):
        c.q.mul_(0.75)
        torch.cuda.synchronize()
        replay.launch()
        device.synchronize()
        c.against()
    replay.destroy()
    plan.destroy()


def refused(match, call):
    with pytest.raises(hip.CpdeError, match=match) as err:
        call()
    assert err.value.code == hip.EINVAL


def test_refusals(device):
    make = lambda *a, **k: hip.Attention(device, *a, **k)
    refused('element type', lambda: make(7, 1, 8, 8, 2, 2, 32))
    refused('whole number of times', lambda: make(hip.F32, 1, 8, 8, 3, 2, 32))
    refused('1 to 128', lambda: make(hip.F32, 1, 8, 8, 2, 2, 129))
    refused('1 to 128', lambda: make(hip.F32, 1, 8, 8, 2, 2, 0))
    refused('negative size', lambda: make(hip.F32, 1, -1, 8, 2, 2, 32))
    refused('scale', lambda: make(hip.F32, 1, 8, 8, 2, 2, 32, scale=-1.0))
    refused('scale', lambda: make(hip.F32, 1, 8, 8, 2, 2, 32, scale=math.nan))
    refused('scale', lambda: make(hip.F32, 1, 8, 8, 2, 2, 32, scale=1e-35))
    refused('scale', lambda: make(hip.F32, 1, 8, 8, 2, 2, 32, scale=math.inf))
    refused('too many', lambda: make(hip.F32, 1, 1 << 30, 8, 4, 2, 32))
    refused('too many workgroups', lambda: make(hip.F32, 1 << 20, 1 << 20, 8, 2, 2, 32))
    c = Case('f32', 2, 8, 9, 2, 2, 32)
    plan = make(c.type, *c.shape, backward=False)
    q, k, v, out, dout, dq, dk, dv = c.view('q', 'k', 'v', 'out', 'dout', 'dq', 'dk', 'dv')
    refused('without a backward', lambda: plan.backward(q, k, v, out, c.lse, dout, dq, dk, dv))
    refused('null tensor', lambda: plan.forward(hip.Heads(None, 1, 1, 1), k, v, out))
    refused('null argument', lambda: plan.forward(None, k, v, out))
    refused('negative stride', lambda: plan.forward(hip.Heads(q.data, -1, 64, 32), k, v, out))
    refused('overlap', lambda: plan.forward(q, k, v, hip.Heads(out.data, 0, 64, 32)))
    refused('overlap', lambda: plan.forward(q, k, v, hip.Heads(out.data, 512, 64, 16)))
    plan.destroy()
    plan = make(c.type, *c.shape)
    refused('null statistics', lambda: plan.backward(q, k, v, out, None, dout, dq, dk, dv))
    refused('overlap', lambda: plan.backward(q, k, v, out, c.lse, dout, dq, hip.Heads(dk.data, 0, 64, 32), dv))
    device.capture_begin()
    refused('capture', lambda: make(hip.F32, 1, 8, 8, 2, 2, 32))
    device.capture_end(keep=False)
    plan.destroy()
    # nothing is left behind
    c.run(device)
    c.against()
