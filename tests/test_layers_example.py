"""examples/sequence_layers.py without a GPU: what its autograd functions refuse."""
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'examples'))
import sequence_layers as example  # noqa: E402


class Plan:
    """Stands for an operator: its results do not matter here."""

    def forward(self, *args, **kwargs):
        pass

    backward = forward


@pytest.fixture(autouse=True)
def host_tensors(monkeypatch):
    view = SimpleNamespace(of=lambda t: t)
    monkeypatch.setattr(example, 'hip', SimpleNamespace(Rows=view, Heads=view))


def outputs(x):
    """The functions on one input beside a path of torch's own."""
    weight = torch.ones(8, 8)
    yield example.Product.apply(x.view(4, 8), weight, weight[0], x.view(4, 8), Plan(), True).flatten()
    yield example.Product.apply(x.view(4, 8), weight, None, None, Plan(), False).flatten()
    heads = x.view(1, 4, 2, 4)
    yield torch.cat(example.Rotate.apply(heads, heads, weight[0, :4], weight[0, :4], Plan())).flatten()[:32]


@pytest.mark.parametrize('which', [0, 1, 2])
def test_second_derivatives_are_refused(which):
    x = torch.linspace(-1, 1, 32, requires_grad=True)
    loss = (list(outputs(x))[which] + x ** 3).sum()
    with pytest.raises(RuntimeError, match='first derivatives only'):
        torch.autograd.grad(loss, x, create_graph=True)


@pytest.mark.parametrize('which', [0, 1, 2])
def test_first_derivatives_are_not(which):
    x = torch.linspace(-1, 1, 32, requires_grad=True)
    loss = (list(outputs(x))[which] + x ** 3).sum()
    assert torch.autograd.grad(loss, x)[0].shape == x.shape
