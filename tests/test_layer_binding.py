"""What the Python binding of the layer operators checks of tensors before their addresses
go to the library (which is a stub here: no GPU; tensors have no memory)."""
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


def rows(*shape, dtype=torch.bfloat16):
    return hip.Rows.of(tensor(*shape, dtype=dtype))


def refused(calls, cases):
    del calls[:]
    for match, call in cases:
        with pytest.raises(ValueError, match=match):
            call()
    assert not calls


def test_linear(calls):
    plan = hip.Linear(DEVICE, hip.BF16, 50, 24, 40, hip.SILU)
    x, w, y = rows(50, 24), rows(40, 24), rows(50, 40)
    bias = tensor(40)
    plan.forward(50, x, w, y, bias=bias, residual=rows(64, 48), pre=rows(50, 40))
    plan.forward(30, rows(30, 24), w, rows(30, 40))
    plan.forward(30, hip.Rows(4096, 24), hip.Rows(8192, 24), hip.Rows(4096, 40), bias=16384)
    plan.backward(50, x, w, y, pre=y, dx=rows(50, 24), dweight=rows(40, 24), dbias=bias)
    plan.backward(50, None, None, y, pre=y, dbias=bias)
    assert calls[1:] == ['cpde_linear_forward'] * 3 + ['cpde_linear_backward'] * 2
    refused(calls, [
        ('^x has the sizes', lambda: plan.forward(50, rows(49, 24), w, y)),
        ('^x has the sizes', lambda: plan.forward(50, rows(50, 23), w, y)),
        ('^weight has the sizes', lambda: plan.forward(50, x, rows(24, 40), y)),
        ('^y has the sizes', lambda: plan.forward(50, x, w, rows(50, 39))),
        ('^residual has the sizes', lambda: plan.forward(50, x, w, y, residual=rows(50, 24))),
        ('^pre is a tensor of float32', lambda: plan.forward(50, x, w, y, pre=rows(50, 40, dtype=torch.float32))),
        ('^bias is a tensor of float32', lambda: plan.forward(50, x, w, y, bias=tensor(40, dtype=torch.float32))),
        ('^bias is not 40 elements', lambda: plan.forward(50, x, w, y, bias=tensor(39))),
        ('^bias is not 40 elements', lambda: plan.forward(50, x, w, y, bias=tensor(80)[::2])),
        ('^dy has the sizes', lambda: plan.backward(50, x, w, x, pre=y, dx=x)),
        ('^dx has the sizes', lambda: plan.backward(50, x, w, y, pre=y, dx=rows(40, 24))),
        ('^dweight has the sizes', lambda: plan.backward(50, x, w, y, pre=y, dweight=rows(24, 40))),
        ('^dbias is a tensor of float32', lambda: plan.backward(50, x, w, y, pre=y, dbias=tensor(40, dtype=torch.float32)))])


def test_bias_in_a_buffer_is_checked_by_its_bytes():
    plan = hip.Linear(DEVICE, hip.F16, 50, 24, 40)
    buffer = object.__new__(hip.Buffer)
    buffer.nbytes, buffer.ptr = 79, 4096
    x, w, y = (rows(*s, dtype=torch.float16) for s in ((50, 24), (40, 24), (50, 40)))
    with pytest.raises(ValueError, match='^bias has 79 bytes'):
        plan.forward(50, x, w, y, bias=buffer)
    buffer.nbytes = 80
    plan.forward(50, x, w, y, bias=buffer)


def heads(*shape, dtype=torch.bfloat16):
    return hip.Heads.of(tensor(*shape, dtype=dtype))


def test_rotation(calls):
    plan = hip.Rotation(DEVICE, hip.BF16, 2, 5, 4, 2, 32)
    q, k, w = heads(2, 5, 4, 32), heads(2, 5, 2, 32), tensor(32)
    at = tensor(2, 5, dtype=torch.int32)
    plan.forward(q, k, q, heads(2, 90, 2, 32), w, w, at)
    plan.forward(q, k, q, k)
    plan.backward(q, k, q, k, q, k, w, w, w, w, at)
    assert calls[1:] == ['cpde_rotation_forward'] * 2 + ['cpde_rotation_backward']
    refused(calls, [
        ('^q has the sizes', lambda: plan.forward(k, k, q, k)),
        ('^k has the sizes', lambda: plan.forward(q, heads(2, 4, 2, 32), q, k)),
        ('^q_out has the sizes', lambda: plan.forward(q, k, heads(1, 5, 4, 32), k)),
        ('^k_out is a tensor of float32', lambda: plan.forward(q, k, q, heads(2, 5, 2, 32, dtype=torch.float32))),
        ('^q_weight is not 32 elements', lambda: plan.forward(q, k, q, k, tensor(31))),
        ('^k_weight is a tensor of float32', lambda: plan.forward(q, k, q, k, w, tensor(32, dtype=torch.float32))),
        ('^positions is a tensor of int64', lambda: plan.forward(q, k, q, k, positions=tensor(2, 5, dtype=torch.int64))),
        ('^positions is not 10 elements', lambda: plan.forward(q, k, q, k, positions=tensor(2, 4, dtype=torch.int32))),
        ('^dq_out has the sizes', lambda: plan.backward(q, k, k, k, q, k)),
        ('^dk has the sizes', lambda: plan.backward(q, k, q, k, q, heads(2, 5, 1, 32))),
        ('^dq_weight is not 32 elements', lambda: plan.backward(q, k, q, k, q, k, dq_weight=tensor(16)))])


def test_rotation_of_one_side(calls):
    plan = hip.Rotation(DEVICE, hip.BF16, 2, 5, 4, 0, 32)
    q = heads(2, 5, 4, 32)
    plan.forward(q, None, q, None)
    assert calls[-1] == 'cpde_rotation_forward'


def matrices(*shape, dtype=torch.float16):
    return hip.Matrices.of(tensor(*shape, dtype=dtype))


def test_orthogonal(calls):
    plan = hip.Orthogonal(DEVICE, hip.F16, 2, 24, 40)
    x, m = matrices(2, 24, 40), matrices(2, 24, 40, dtype=torch.float32)
    plan.forward(x, matrices(3, 24, 48))
    plan.update(x, m, x, 0.1)
    assert calls[1:] == ['cpde_orthogonal_forward', 'cpde_orthogonal_update']
    refused(calls, [
        ('^x has the sizes', lambda: plan.forward(matrices(1, 24, 40), x)),
        ('^out has the sizes', lambda: plan.forward(x, matrices(2, 40, 24))),
        ('^x is a tensor of float32', lambda: plan.forward(m, x)),
        ('^momentum is a tensor of float16', lambda: plan.update(x, x, x, 0.1)),
        ('^momentum has the sizes', lambda: plan.update(x, matrices(2, 23, 40, dtype=torch.float32), x, 0.1)),
        ('^gradient is a tensor of float32', lambda: plan.update(m, m, x, 0.1)),
        ('^weight has the sizes', lambda: plan.update(x, m, matrices(2, 24, 39), 0.1))])


def test_tensors_that_have_no_view():
    with pytest.raises(ValueError, match='not contiguous'):
        hip.Matrices.of(tensor(2, 24, 40).transpose(1, 2))
    with pytest.raises(ValueError, match='not on a GPU'):
        hip.Matrices.of(torch.empty(2, 3, 4))
