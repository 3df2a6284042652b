"""A network that continues a PDE's solution in time: the layer operators in use.

    python examples/sequence_layers.py [--steps 300]

Advection with diffusion, u_t + c u_x = nu u_xx, on a ring: a sequence's tokens are
the values of u on a grid at times one step apart, with a speed c of its own, and the
network gives each token's next one.  Its layer is the framework's operators: products
with their bias, activation and residual, each head's norm and rotation by the token's
place, causal attention; its matrices are moved along orthogonalised momenta and what is
left (biases, norms' weights, the first and last matrices) by torch's Adam.
"""
import argparse
import math
import sys
from pathlib import Path

import torch

sys.path[:0] = [str(Path(__file__).resolve().parents[1]), str(Path(__file__).resolve().parent)]
from cpde_amd import hip  # noqa: E402
from sequence_model import Attend, once  # noqa: E402

GRID, DIFFUSIVITY, STEP = 16, 0.02, 0.1


class Product(torch.autograd.Function):
    """activation(x W^T + bias) + residual over x's rows; bias and residual may be None."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, plan, bent):
        # (columns that repeat a value have a stride of zero)
        rows = x.reshape(-1, x.shape[-1]).contiguous()
        residual = None if residual is None else residual.reshape(-1, weight.shape[0]).contiguous()
        y = torch.empty((rows.shape[0], weight.shape[0]), device=x.device, dtype=x.dtype)
        pre = torch.empty_like(y) if bent else None
        plan.forward(rows.shape[0], hip.Rows.of(rows), hip.Rows.of(weight), hip.Rows.of(y), bias=bias,
                     residual=None if residual is None else hip.Rows.of(residual),
                     pre=None if pre is None else hip.Rows.of(pre))
        ctx.plan, ctx.shape = plan, x.shape
        ctx.save_for_backward(rows, weight, pre)
        return y.view(*x.shape[:-1], -1)

    @staticmethod
    @once
    def backward(ctx, dy):
        rows, weight, pre = ctx.saved_tensors
        flat = dy.reshape(rows.shape[0], -1).contiguous()  # (a sum's gradient repeats one value)
        dx, dweight = (torch.empty_like(t) if n else None for t, n in zip((rows, weight), ctx.needs_input_grad))
        dbias = torch.empty(weight.shape[0], device=dy.device, dtype=dy.dtype) if ctx.needs_input_grad[2] else None
        ctx.plan.backward(rows.shape[0], hip.Rows.of(rows), hip.Rows.of(weight), hip.Rows.of(flat),
                          pre=None if pre is None else hip.Rows.of(pre), dx=None if dx is None else hip.Rows.of(dx),
                          dweight=None if dweight is None else hip.Rows.of(dweight), dbias=dbias)
        return (None if dx is None else dx.view(ctx.shape), dweight, dbias, dy if ctx.needs_input_grad[3] else None, None,
                None)


class Rotate(torch.autograd.Function):
    """Queries and keys [batch, tokens, heads, width]: each head's norm, and its rotation."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, plan):
        q, k = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k))
        q_out, k_out = torch.empty(q.shape, device=q.device), torch.empty(k.shape, device=k.device)
        plan.forward(*(hip.Heads.of(t) for t in (q, k, q_out, k_out)), q_weight, k_weight)
        ctx.plan = plan
        ctx.save_for_backward(q, k, q_weight, k_weight)
        return q_out, k_out

    @staticmethod
    @once
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight = ctx.saved_tensors
        dq_out, dk_out = dq_out.contiguous(), dk_out.contiguous()
        dq, dk = torch.empty(q.shape, device=q.device), torch.empty(k.shape, device=k.device)
        dq_weight, dk_weight = torch.empty_like(q_weight), torch.empty_like(k_weight)
        ctx.plan.backward(*(hip.Heads.of(t) for t in (q, k, dq_out, dk_out, dq, dk)), q_weight, k_weight, dq_weight,
                          dk_weight)
        return dq, dk, dq_weight, dk_weight, None


class LayerModel(torch.nn.Module):
    def __init__(self, device, batch, tokens, width=64, heads=4, seed=1):
        super().__init__()
        generator = torch.Generator().manual_seed(seed)

        def weights(outputs, inputs):
            return torch.nn.Parameter((torch.randn((outputs, inputs), generator=generator) / math.sqrt(inputs)).cuda())

        def values(n, value):
            return torch.nn.Parameter(torch.full((n,), value, device='cuda'))

        self.width, self.heads = width, heads
        dim = width // heads
        self.first, self.last = weights(width, GRID), weights(GRID, width)
        self.attended, self.joined = weights(3 * width, width), weights(width, width)
        self.up, self.down = weights(2 * width, width), weights(width, 2 * width)
        self.up_bias, self.down_bias = values(2 * width, 0.0), values(width, 0.0)
        self.q_weight, self.k_weight = values(dim, 1.0), values(dim, 1.0)
        rows = batch * tokens
        self.plans = {n: hip.Linear(device, hip.F32, rows, *reversed(getattr(self, n).shape), activation)
                      for n, activation in (('first', hip.NONE), ('attended', hip.NONE), ('joined', hip.NONE), ('up', hip.GELU),
                                            ('down', hip.NONE), ('last', hip.NONE))}
        self.rotation = hip.Rotation(device, hip.F32, batch, tokens, heads, heads, dim)
        self.attention = hip.Attention(device, hip.F32, batch, tokens, tokens, heads, heads, dim, right=0)

    def product(self, name, x, bias=None, residual=None):
        return Product.apply(x, getattr(self, name), bias, residual, self.plans[name], name == 'up')

    def forward(self, u):
        x = self.product('first', u)
        q, k, v = (t.unflatten(-1, (self.heads, -1)) for t in self.product('attended', x).split(self.width, -1))
        q, k = Rotate.apply(q, k, self.q_weight, self.k_weight, self.rotation)
        x = self.product('joined', Attend.apply(q, k, v, self.attention).flatten(2), residual=x)
        x = self.product('down', self.product('up', x, self.up_bias), self.down_bias, residual=x)
        return self.product('last', x, residual=u)

    def destroy(self):
        for plan in (*self.plans.values(), self.rotation, self.attention):
            plan.destroy()


class Orthogonalised:
    """The step of `matrices` along their orthogonalised momenta."""

    def __init__(self, device, matrices, rate):
        self.matrices, self.rate = list(matrices), rate
        self.momenta = [torch.zeros_like(w) for w in self.matrices]
        self.plans = {w.shape: hip.Orthogonal(device, hip.F32, 1, *w.shape) for w in self.matrices}

    @torch.no_grad()
    def step(self):
        for w, m in zip(self.matrices, self.momenta):
            view = [hip.Matrices.of(t[None]) for t in (w.grad, m, w)]
            self.plans[w.shape].update(*view, self.rate)

    def destroy(self):
        for plan in self.plans.values():
            plan.destroy()


def problem(batch, tokens, generator):
    """States (batch, tokens + 1, GRID) of u, each sequence with a speed of its own."""
    k = torch.arange(1, 4, device='cuda', dtype=torch.float32)
    a, phase = torch.rand((2, batch, 1, 1, 3), generator=generator, device='cuda')
    speed = 2 * torch.rand((batch, 1, 1, 1), generator=generator, device='cuda') - 1
    t = STEP * torch.arange(tokens + 1, device='cuda')[:, None, None]
    x = torch.arange(GRID, device='cuda')[:, None] * (2 * math.pi / GRID)
    return (a * torch.exp(-DIFFUSIVITY * k * k * t) * torch.sin(k * (x - speed * t) + 2 * math.pi * phase)).sum(-1)


def train(steps=300, batch=16, tokens=32, rate=0.02, report=None):
    """Losses of the steps."""
    device = hip.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    model = LayerModel(device, batch, tokens)
    inner = [model.attended, model.joined, model.up, model.down]
    orthogonal = Orthogonalised(device, inner, rate)
    others = [p for p in model.parameters() if all(p is not w for w in inner)]
    adam = torch.optim.Adam(others, 3e-3)
    generator = torch.Generator('cuda').manual_seed(2)
    losses = []
    for step in range(steps):
        u = problem(batch, tokens, generator)
        loss = ((model(u[:, :-1]) - u[:, 1:]) ** 2).mean()
        model.zero_grad()
        loss.backward()
        orthogonal.step()
        adam.step()
        losses.append(loss.detach())
        if report and (step % 50 == 0 or step == steps - 1):
            report(f'step {step}: mean squared error {loss.item():.6f}')
    losses = torch.stack(losses).tolist()
    orthogonal.destroy()
    model.destroy()
    device.close()
    return losses


if __name__ == '__main__':
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument('--steps', type=int, default=300)
    train(parser.parse_args().steps, report=lambda line: print(line, flush=True))
