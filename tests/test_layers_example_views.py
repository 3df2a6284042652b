"""examples/sequence_layers.py without a GPU: what its autograd functions hand to the
operators, whatever their inputs and incoming gradients repeat."""
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'examples'))
import sequence_layers as example  # noqa: E402


class Plan:
    """Stands for an operator and keeps what its gradient was asked for."""
    asked = None

    def forward(self, *args, **kwargs):
        pass

    def backward(self, *args, **kwargs):
        self.asked = {n for n in ('dx', 'dweight', 'dbias') if kwargs.get(n) is not None}


@pytest.fixture(autouse=True)
def host_tensors(monkeypatch):
    def of(t):
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise ValueError('the last axis is not contiguous')
        return t

    view = SimpleNamespace(of=of)
    monkeypatch.setattr(example, 'hip', SimpleNamespace(Rows=view, Heads=view))


def leaf(*shape, grad=True):
    return torch.ones(shape, requires_grad=grad)


def test_gradients_that_repeat_a_value():
    """The gradient of a sum has strides of zero."""
    for bent in (False, True):
        x, w, b, r = leaf(2, 3, 8), leaf(4, 8), leaf(4), leaf(2, 3, 4)
        plan = Plan()
        example.Product.apply(x, w, b, r, plan, bent).sum().backward()
        assert plan.asked == {'dx', 'dweight', 'dbias'}
        assert [t.grad.shape for t in (x, w, b, r)] == [t.shape for t in (x, w, b, r)]
        assert (r.grad == 1).all()


def test_inputs_that_repeat_a_column():
    x, r = leaf(2, 3, 1).expand(2, 3, 8), leaf(2, 3, 1).expand(2, 3, 4)
    w = leaf(4, 8)
    plan = Plan()
    example.Product.apply(x, w, None, r, plan, False).sum().backward()
    assert plan.asked == {'dx', 'dweight'}
    q, k = leaf(1, 3, 2, 1).expand(1, 3, 2, 8), leaf(1, 3, 2, 1).expand(1, 3, 2, 8)
    sum(t.sum() for t in example.Rotate.apply(q, k, leaf(8), leaf(8), plan)).backward()


@pytest.mark.parametrize('needed', range(1, 16))
def test_only_gradients_that_are_needed(needed):
    """What no gradient is asked of costs no product."""
    has = [bool(needed >> i & 1) for i in range(4)]
    shapes = (3, 8), (4, 8), (4,), (3, 4)
    x, w, b, r = leaves = [leaf(*s, grad=h) for s, h in zip(shapes, has)]
    plan = Plan()
    example.Product.apply(x, w, b, r, plan, True).sum().backward()
    assert (plan.asked or set()) == {n for n, h in zip(('dx', 'dweight', 'dbias'), has) if h}
    assert [t.grad is not None for t in leaves] == has
