"""What the Python binding of the operators on sequences checks of tensors before their
addresses go to the library (which is a stub here: no GPU; tensors have no memory)."""
from types import SimpleNamespace

import pytest
import torch

from cpde_amd import hip


@pytest.fixture(autouse=True)
def calls(monkeypatch):
    """Names of the library's entry points that were reached."""
    made = []

    class Stub:
        def __getattr__(self, name):
            return lambda *args: made.append(name) or hip.OK

    monkeypatch.setattr(hip, 'load', lambda: Stub())
    return made


# the device of torch's tensors without memory (their number is -1)
DEVICE = SimpleNamespace(handle=None, ordinal=-1)


def tensor(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device='meta')


def attention_views(batch=2, queries=5, keys=7, heads=4, kv_heads=2, dim=32, **other):
    sizes = {n: (batch, queries, heads, dim) for n in ('q', 'out', 'dout', 'dq')}
    sizes.update({n: (batch, keys, kv_heads, dim) for n in ('k', 'v', 'dk', 'dv')})
    views = {n: hip.Heads.of(tensor(*other.get(n, shape), dtype=other.get(n + '_type', torch.bfloat16)))
             for n, shape in sizes.items()}
    views['lse'] = other.get('lse', tensor(batch, heads, queries, dtype=torch.float32))
    return views


def forward(v, **lengths):
    plan = hip.Attention(DEVICE, hip.BF16, 2, 5, 7, 4, 2, 32)
    plan.forward(v['q'], v['k'], v['v'], v['out'], v['lse'], **lengths)


def backward(v, **lengths):
    plan = hip.Attention(DEVICE, hip.BF16, 2, 5, 7, 4, 2, 32)
    plan.backward(*(v[n] for n in ('q', 'k', 'v', 'out', 'lse', 'dout', 'dq', 'dk', 'dv')), **lengths)


def test_fitting_tensors_pass(calls):
    lengths = tensor(2, dtype=torch.int32)
    forward(attention_views(), query_lengths=lengths, key_lengths=lengths)
    backward(attention_views(), query_lengths=lengths, key_lengths=lengths)
    # larger ones (a cache with room), views of bare addresses, addresses
    forward(attention_views(k=(3, 90, 2, 32), v=(3, 90, 2, 64)))
    v = attention_views(lse=4096)
    v['q'] = hip.Heads(4096, 1, 1, 1)
    forward(v, key_lengths=8192)
    forward(attention_views(lse=None))
    assert calls.count('cpde_attention_forward') == 4 and calls.count('cpde_attention_backward') == 1


@pytest.mark.parametrize('name,shape', [
    ('q', (2, 4, 4, 32)), ('q', (1, 5, 4, 32)), ('k', (2, 6, 2, 32)), ('v', (2, 7, 1, 32)), ('out', (2, 5, 4, 31)),
    ('dout', (2, 5, 3, 32)), ('dq', (2, 4, 4, 32)), ('dk', (2, 6, 2, 32)), ('dv', (2, 7, 2, 16))])
def test_attention_refuses_smaller_tensors(calls, name, shape):
    with pytest.raises(ValueError, match=f'^{name} has the sizes'):
        (backward if name.startswith('d') else forward)(attention_views(**{name: shape}))
    assert not any('ward' in c for c in calls)


@pytest.mark.parametrize('name', ['q', 'k', 'v', 'out', 'dout', 'dq', 'dk', 'dv'])
def test_attention_refuses_other_types(calls, name):
    with pytest.raises(ValueError, match=f'^{name} is a tensor of float32'):
        (backward if name.startswith('d') else forward)(attention_views(**{name + '_type': torch.float32}))
    assert not any('ward' in c for c in calls)


def test_attention_refuses_unfit_lists(calls):
    for call in (forward, backward):
        with pytest.raises(ValueError, match='^lse is a tensor of bfloat16'):
            call(attention_views(lse=tensor(2, 4, 5)))
        with pytest.raises(ValueError, match='^lse is not 40 elements'):
            call(attention_views(lse=tensor(2, 4, 4, dtype=torch.float32)))
        with pytest.raises(ValueError, match='^lse is not 40 elements'):
            call(attention_views(lse=tensor(2, 5, 4, dtype=torch.float32).transpose(1, 2)))
        for name in ('query_lengths', 'key_lengths'):
            with pytest.raises(ValueError, match=f'^{name} is a tensor of int64'):
                call(attention_views(), **{name: tensor(2, dtype=torch.int64)})
            with pytest.raises(ValueError, match=f'^{name} is not 2 elements'):
                call(attention_views(), **{name: tensor(1, dtype=torch.int32)})
    assert not any('ward' in c for c in calls)


def test_tensors_of_the_host_are_refused(calls):
    plan = hip.Embedding(SimpleNamespace(handle=None, ordinal=0), hip.F16, 100, 24, 50)
    with pytest.raises(ValueError, match='^ids is a tensor of int32 on cpu'):
        plan.forward(torch.zeros(50, dtype=torch.int32), 50, hip.Rows(4096, 24), hip.Rows(8192, 24))
    assert 'cpde_embedding_forward' not in calls
    with pytest.raises(ValueError, match='not on a GPU'):
        hip.Heads.of(torch.empty(1, 2, 3, 4))
    with pytest.raises(ValueError, match='not on a GPU'):
        hip.Rows.of(torch.empty(3, 4))


def test_other_gpus_tensors_are_refused(calls):
    v = attention_views()
    v['k'].held = ('bfloat16', 1, *v['k'].held[2:])
    with pytest.raises(ValueError, match='^k is a tensor of bfloat16 on GPU 1'):
        forward(v)
    assert 'cpde_attention_forward' not in calls


def rows(*shape, dtype=torch.float16):
    return hip.Rows.of(tensor(*shape, dtype=dtype))


def test_embedding(calls):
    plan = hip.Embedding(DEVICE, hip.F16, 100, 24, 50, index_bytes=8)
    ids = tensor(50, dtype=torch.int64)
    table, out, dtable = rows(100, 24), rows(50, 24), rows(100, 24, dtype=torch.float32)
    plan.forward(ids, 50, table, out)
    plan.backward(ids, 40, rows(40, 24), dtable)
    assert calls[-2:] == ['cpde_embedding_forward', 'cpde_embedding_backward']
    del calls[:]
    for match, call in (
            ('^ids is a tensor of int32', lambda: plan.forward(tensor(50, dtype=torch.int32), 50, table, out)),
            ('^ids is not 50', lambda: plan.forward(tensor(49, dtype=torch.int64), 50, table, out)),
            ('^ids is not 25', lambda: plan.forward(tensor(50, dtype=torch.int64)[::2], 25, table, out)),
            ('^table has the sizes', lambda: plan.forward(ids, 50, rows(99, 24), out)),
            ('^table is a tensor of float32', lambda: plan.forward(ids, 50, dtable, out)),
            ('^out has the sizes', lambda: plan.forward(ids, 50, table, rows(49, 24))),
            ('^dout has the sizes', lambda: plan.backward(ids, 50, rows(50, 23), dtable)),
            ('^dtable is a tensor of float16', lambda: plan.backward(ids, 50, out, table)),
            ('^dtable has the sizes', lambda: plan.backward(ids, 50, out, rows(99, 24, dtype=torch.float32)))):
        with pytest.raises(ValueError, match=match):
            call()
    assert not calls


def test_dropout(calls):
    device = object.__new__(hip.Device)
    device.handle, device.ordinal = None, -1
    x = rows(8, 16)
    device.dropout(hip.F16, 8, 16, x, rows(9, 16), 0.5, 1, residual=hip.Rows(4096, 16))
    assert calls == ['cpde_dropout']
    for match, call in (
            ('^x is a tensor', lambda: device.dropout(hip.BF16, 8, 16, x, x, 0.5, 1)),
            ('^y has the sizes', lambda: device.dropout(hip.F16, 8, 16, x, rows(7, 16), 0.5, 1)),
            ('^residual has the sizes', lambda: device.dropout(hip.F16, 8, 16, x, x, 0.5, 1, residual=rows(8, 15)))):
        with pytest.raises(ValueError, match=match):
            call()
    assert calls == ['cpde_dropout']
