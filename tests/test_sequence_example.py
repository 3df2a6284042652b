"""examples/sequence_model.py without a GPU: what its autograd functions refuse."""
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'examples'))
import sequence_model as example  # noqa: E402


class Plan:
    """Stands for an operator: its results do not matter here."""

    def forward(self, *args, **kwargs):
        pass

    backward = dropout = forward


@pytest.fixture(autouse=True)
def host_tensors(monkeypatch):
    views = SimpleNamespace(of=lambda t: t)
    monkeypatch.setattr(example, 'hip', SimpleNamespace(F32=0, Heads=views, Rows=lambda *a: a))
    example.hip.Rows.of = views.of


def outputs(x):
    """The three functions on one input beside a path of torch's own."""
    heads = x.view(1, 4, 2, 4)
    yield example.Attend.apply(heads, heads, heads, Plan()).flatten()
    yield example.Lookup.apply(x.view(4, 8), torch.zeros(4, dtype=torch.int64), Plan(), 1.0).flatten()
    yield example.Dropout.apply(x, x, Plan(), 0.5, 1, 0)


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
