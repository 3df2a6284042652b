"""examples/sequence_model.py: the operators together in a network that is trained."""
import sys
from pathlib import Path

import pytest
import torch

from cpde_amd import hip
from sequences import keep

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'examples'))
import sequence_model as example  # noqa: E402

pytestmark = pytest.mark.gpu


def plain_forward(model, ids, points, masks):
    """The same network in float64 by torch alone, on the masks of its dropouts."""
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in model.named_parameters()}
    masks = iter(masks)

    def attend(q, k, v):
        q, k, v = (t.view(*t.shape[:-1], model.heads, -1).transpose(1, 2) for t in (q, k, v))
        weight = torch.softmax(torch.matmul(q, k.transpose(2, 3)) * q.shape[-1] ** -0.5, -1)
        return torch.matmul(weight, v).transpose(1, 2).flatten(2)

    def dropout(x, residual):
        mask, up = next(masks)
        return torch.where(mask.view(x.shape), x * up, 0.0) + residual

    x = p['table'][ids.cpu()] * 8.0
    x = dropout(attend(*(x @ p['tokens_in']).split(model.width, -1)), x)
    points = points.cpu().double()
    location = torch.cat([points, torch.sin(torch.pi * points)], -1) @ p['points_in']
    y = dropout(attend(location @ p['reads'], *(x @ p['read_by']).split(model.width, -1)), location)
    return (torch.sigmoid(y @ p['hidden']) @ p['out']).squeeze(-1), p


def test_gradients_of_the_whole_network():
    """One step with dropout against float64: parameters' gradients to 1e-4 of their norm
    (a float network of six products and two attentions; its sums of up to 2,000
    terms carry some 1e-6)."""
    batch, points = 4, 21
    device = hip.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    model = example.SequenceModel(device, batch, points, probability=0.25)
    ids, at, u = example.problem(batch, points, torch.Generator('cuda').manual_seed(7))
    loss = ((model(ids, at) - u) ** 2).mean()
    loss.backward()
    up, masks, offset = 2.0 ** 32 / (2.0 ** 32 - round(0.25 * 2 ** 32)), [], 0
    for count in (batch * example.MODES * model.width, batch * points * model.width):
        masks.append((keep(1, count, 0.25, model.seed, offset)[0], up))
        offset += (count + 3) // 4
    want, p = plain_forward(model, ids, at, masks)
    want_loss = ((want - u.cpu().double()) ** 2).mean()
    want_loss.backward()
    assert abs(loss.item() / want_loss.item() - 1) < 1e-5
    for name, t in model.named_parameters():
        far = float((t.grad.cpu().double() - p[name].grad).norm() / p[name].grad.norm())
        assert far < 1e-4, (name, far)
    model.destroy()
    device.close()


def test_training_learns():
    losses = example.train(steps=200)
    first, last = sum(losses[:10]) / 10, sum(losses[-20:]) / 20
    print(f'[result] mean squared error {first:.4f} -> {last:.4f}', flush=True)
    assert last < first / 3
