"""examples/sequence_layers.py: the layer operators and attention together in a network
that is trained."""
import math
import sys
from pathlib import Path

import pytest
import torch

from cpde_amd import hip
from layers import orthogonal

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'examples'))
import sequence_layers as example  # noqa: E402

pytestmark = pytest.mark.gpu


def plain_forward(model, u):
    """The same network in float64 by torch alone."""
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in model.named_parameters()}
    u = u.detach().cpu().double()
    batch, tokens = u.shape[:2]
    dim = model.width // model.heads
    angle = torch.arange(tokens, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)

    def rotate(x, weight):
        x = x.unflatten(-1, (model.heads, dim))
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
        a, b = x.split(dim // 2, -1)
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        return torch.cat([a * c - b * s, a * s + b * c], -1).transpose(1, 2)

    x = u @ p['first'].T
    q, k, v = (x @ p['attended'].T).split(model.width, -1)
    q, k = rotate(q, p['q_weight']), rotate(k, p['k_weight'])
    v = v.unflatten(-1, (model.heads, dim)).transpose(1, 2)
    score = torch.matmul(q, k.transpose(2, 3)) * dim ** -0.5
    score = score.masked_fill(torch.ones(tokens, tokens, dtype=torch.bool).triu(1), -math.inf)
    y = torch.matmul(torch.softmax(score, -1), v).transpose(1, 2).flatten(2)
    x = y @ p['joined'].T + x
    z = torch.nn.functional.gelu(x @ p['up'].T + p['up_bias'])
    x = z @ p['down'].T + p['down_bias'] + x
    return x @ p['last'].T + u, p


def test_gradients_of_the_whole_network():
    """One step against float64: parameters' gradients to 1e-4 of their norm (a float network of
    six products, rotations and attention; its sums of up to 1,000 terms carry some 1e-6)."""
    batch, tokens = 5, 21
    device = hip.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    model = example.LayerModel(device, batch, tokens)
    u = example.problem(batch, tokens, torch.Generator('cuda').manual_seed(7))
    loss = ((model(u[:, :-1]) - u[:, 1:]) ** 2).mean()
    loss.backward()
    want, p = plain_forward(model, u[:, :-1])
    want_loss = ((want - u[:, 1:].cpu().double()) ** 2).mean()
    want_loss.backward()
    assert abs(loss.item() / want_loss.item() - 1) < 1e-5
    for name, t in model.named_parameters():
        far = float((t.grad.cpu().double() - p[name].grad).norm() / p[name].grad.norm())
        assert far < 1e-4, (name, far)
    # and the step of its matrices, from momenta of zero
    optimizer = example.Orthogonalised(device, [model.up, model.joined], 0.05)
    before = [t.detach().clone().double() for t in (model.up, model.joined)]
    optimizer.step()
    for w, t in zip(before, (model.up, model.joined)):
        size = 0.05 * math.sqrt(max(1, t.shape[0] / t.shape[1]))
        step = orthogonal(t.grad[None] * 1.95, 5)[0]  # gradient + 0.95 momentum, which is the gradient
        # (five steps of float products on gradients of low rank: 485 times their 2^-22 at most)
        far = float((t.detach().double() - (w - size * step)).norm() / (size * step.norm()))
        assert far < 485 * 2.0 ** -20, far
    optimizer.destroy()
    model.destroy()
    device.close()


def test_training_runs():
    losses = example.train(steps=30)
    print(f'[result] mean squared error {losses[0]:.5f} -> {losses[-1]:.5f}', flush=True)
    assert len(losses) == 30 and all(math.isfinite(x) for x in losses)
