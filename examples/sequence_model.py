"""A network that reads a PDE's data as a sequence: the operators on sequences in use.

    python examples/sequence_model.py [--steps 300]

The heat equation on (0, 1) with u(x, 0) = sum_k a_k sin(k pi x), every a_k one of 16
levels, has u(x, t) = sum_k a_k exp(-(k pi)^2 nu t) sin(k pi x).  The network is given
the levels as tokens and points (x, t), and learns u there: tokens are looked up in a
table (its rows learned), attend to one another, are read by the points, each read
with dropout and added onto what it read for.  The linear layers between are torch's;
a device opened on torch's stream keeps both sides' work in order.
"""
import argparse
import functools
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from cpde_amd import hip  # noqa: E402

MODES, LEVELS, DIFFUSIVITY = 8, 16, 0.05


def once(backward):
    """Gradients come from kernels that autograd does not see into: asked for with
    create_graph=True, whose second derivatives would silently lack their share (torch's
    once_differentiable lets that pass where the incoming gradient is a constant), they
    are refused."""
    @functools.wraps(backward)
    def checked(ctx, *grads):
        if torch.is_grad_enabled():
            raise RuntimeError('the operators on sequences have first derivatives only (create_graph=True)')
        return backward(ctx, *grads)
    return checked


class Lookup(torch.autograd.Function):
    """Rows of the table at the tokens, scaled."""

    @staticmethod
    def forward(ctx, table, ids, plan, scale):
        ctx.plan, ctx.scale, ctx.rows = plan, scale, table.shape[0]
        ctx.save_for_backward(ids)
        out = torch.empty((ids.numel(), table.shape[1]), device=table.device)
        plan.forward(ids, ids.numel(), hip.Rows.of(table), hip.Rows.of(out), scale)
        return out.view(*ids.shape, -1)

    @staticmethod
    @once
    def backward(ctx, dout):
        ids, = ctx.saved_tensors
        dout = dout.reshape(ids.numel(), -1).contiguous()
        dtable = torch.empty((ctx.rows, dout.shape[1]), device=dout.device)
        ctx.plan.backward(ids, ids.numel(), hip.Rows.of(dout), hip.Rows.of(dtable), ctx.scale)
        return dtable, None, None, None


class Attend(torch.autograd.Function):
    """Attention of tensors [batch, tokens, heads, width] of any strides."""

    @staticmethod
    def forward(ctx, q, k, v, plan):
        out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), device=q.device)
        plan.forward(*(hip.Heads.of(t) for t in (q, k, v, out)), lse)
        ctx.plan = plan
        ctx.save_for_backward(q, k, v, out, lse)
        return out

    @staticmethod
    @once
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        dout = dout.contiguous()
        grads = [torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v)]
        ctx.plan.backward(*(hip.Heads.of(t) for t in (q, k, v, out)), lse, hip.Heads.of(dout),
                          *(hip.Heads.of(t) for t in grads))
        return *grads, None


class Dropout(torch.autograd.Function):
    """dropout(x) + residual; the mask is made again for the gradient."""

    @staticmethod
    def forward(ctx, x, residual, device, probability, seed, offset):
        ctx.args = device, probability, seed, offset
        x, residual = x.contiguous(), residual.contiguous()
        y = torch.empty_like(x)
        device.dropout(hip.F32, 1, x.numel(), *(hip.Rows(t.data_ptr(), t.numel()) for t in (x, y)), probability, seed,
                       offset, residual=hip.Rows(residual.data_ptr(), residual.numel()))
        return y

    @staticmethod
    @once
    def backward(ctx, dy):
        device, probability, seed, offset = ctx.args
        dy = dy.contiguous()
        dx = torch.empty_like(dy)
        device.dropout(hip.F32, 1, dy.numel(), *(hip.Rows(t.data_ptr(), t.numel()) for t in (dy, dx)), probability, seed,
                       offset)
        return dx, dy, None, None, None, None


class SequenceModel(torch.nn.Module):
    def __init__(self, device, batch, points, width=64, heads=4, probability=0.05, seed=1):
        super().__init__()
        generator = torch.Generator().manual_seed(seed)

        def weights(*shape):
            return torch.nn.Parameter((torch.randn(shape, generator=generator) / math.sqrt(shape[0])).cuda())

        self.device, self.width, self.heads, self.probability, self.seed = device, width, heads, probability, seed
        self.table = torch.nn.Parameter((0.125 * torch.randn(MODES * LEVELS, width, generator=generator)).cuda())
        self.tokens_in, self.points_in = weights(width, 3 * width), weights(4, width)
        self.reads, self.read_by = weights(width, width), weights(width, 2 * width)
        self.hidden, self.out = weights(width, 2 * width), weights(2 * width, 1)
        self.offset = 0    # of the generator: every call takes counters of its own
        dim = width // heads
        self.lookup = hip.Embedding(device, hip.F32, MODES * LEVELS, width, batch * MODES, index_bytes=8)
        self.among = hip.Attention(device, hip.F32, batch, MODES, MODES, heads, heads, dim)
        self.across = hip.Attention(device, hip.F32, batch, points, MODES, heads, heads, dim)

    def split(self, x):
        return x.view(*x.shape[:-1], self.heads, -1)

    def dropout(self, x, residual):
        probability = self.probability if self.training else 0.0
        y = Dropout.apply(x, residual, self.device, probability, self.seed, self.offset)
        self.offset += (x.numel() + 3) // 4
        return y

    def forward(self, ids, points):
        x = Lookup.apply(self.table, ids, self.lookup, 8.0)
        q, k, v = (self.split(t) for t in (x @ self.tokens_in).split(self.width, -1))
        x = self.dropout(Attend.apply(q, k, v, self.among).flatten(2), x)
        location = torch.cat([points, torch.sin(math.pi * points)], -1) @ self.points_in
        k, v = (self.split(t) for t in (x @ self.read_by).split(self.width, -1))
        y = Attend.apply(self.split(location @ self.reads), k, v, self.across).flatten(2)
        y = self.dropout(y, location)
        return (torch.sigmoid(y @ self.hidden) @ self.out).squeeze(-1)

    def destroy(self):
        for plan in (self.lookup, self.among, self.across):
            plan.destroy()


def problem(batch, points, generator):
    """Levels as tokens (batch, MODES), points (batch, points, 2) and u there."""
    level = torch.randint(0, LEVELS, (batch, MODES), generator=generator, device='cuda')
    k = torch.arange(1, MODES + 1, device='cuda', dtype=torch.float32)
    x, t = torch.rand((2, batch, points, 1), generator=generator, device='cuda')
    a = (level - (LEVELS - 1) / 2) / (LEVELS / 2) / k
    u = (a[:, None] * torch.exp(-(k * math.pi) ** 2 * DIFFUSIVITY * t) * torch.sin(k * math.pi * x)).sum(-1)
    return (k.long() - 1) * LEVELS + level, torch.cat([x, t], -1), u


def train(steps=300, batch=32, points=64, rate=3e-3, report=None):
    """Losses of the steps."""
    device = hip.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    model = SequenceModel(device, batch, points)
    optimizer = torch.optim.Adam(model.parameters(), rate)
    generator = torch.Generator('cuda').manual_seed(2)
    losses = []
    for step in range(steps):
        ids, at, u = problem(batch, points, generator)
        loss = ((model(ids, at) - u) ** 2).mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if report and (step % 50 == 0 or step == steps - 1):
            report(f'step {step}: mean squared error {loss.item():.5f}')
    losses = torch.stack(losses).tolist()
    model.destroy()
    device.close()
    return losses


if __name__ == '__main__':
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument('--steps', type=int, default=300)
    train(parser.parse_args().steps, report=lambda line: print(line, flush=True))
