"""The operators on sequences in float64 (torch, on the host), with bounds on how
far a kernel's results may lie from them.

Bounds are worst cases of the kernels' own steps, first order, element by element:
u is half a unit in the last place of the tensors' type (results and, where matrix
instructions multiply them, probabilities and score gradients are rounded to it
once), e = 2^-24 that of the float sums, and `tiny` where roundings become absolute:
the spacing of f16's smallest values, and float's least normal value, below which
exponentials are zeros."""
import math

import numpy as np
import torch

from cpde_amd import hip

TYPES = {'f32': (torch.float32, hip.F32), 'f16': (torch.float16, hip.F16), 'bf16': (torch.bfloat16, hip.BF16)}
UNIT = {'f32': 2.0 ** -24, 'f16': 2.0 ** -11, 'bf16': 2.0 ** -8}
LEAST = 2.0 ** -126
TINY = {'f32': LEAST, 'f16': 2.0 ** -24, 'bf16': LEAST}
E = 2.0 ** -24


def visible(ql, kl, lq, lk, left, right):
    """(lq, lk): which keys each query sees."""
    i, j = torch.arange(lq)[:, None], torch.arange(lk)[None, :]
    at = j - (i + kl - ql)
    seen = (i < ql) & (j < kl)
    if left >= 0:
        seen &= at >= -left
    if right >= 0:
        seen &= at <= right
    return seen


def attention(q, k, v, scale, left=-1, right=-1, query_lengths=None, key_lengths=None, dout=None, dtype='f32'):
    """{name: (values, bounds)} of out, lse and (with dout) dq, dk, dv; tensors [batch][token][head][dim]."""
    u, tiny = UNIT[dtype], TINY[dtype]
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    batch, lq, heads, dim = q.shape
    lk, group = k.shape[1], heads // k.shape[2]
    names = ['out', 'lse'] + (['dq', 'dk', 'dv'] if dout is not None else [])
    shapes = {'out': q.shape, 'lse': (batch, heads, lq), 'dq': q.shape, 'dk': k.shape, 'dv': v.shape}
    want = {n: torch.zeros(shapes[n], dtype=torch.float64) for n in names}
    far = {n: torch.zeros(shapes[n], dtype=torch.float64) for n in names}
    do = dout.detach().cpu().double() if dout is not None else None
    for b in range(batch):
        ql = lq if query_lengths is None else min(max(int(query_lengths[b]), 0), lq)
        kl = lk if key_lengths is None else min(max(int(key_lengths[b]), 0), lk)
        # (what lies past the lengths is not to be read)
        keys = [torch.where((torch.arange(lk) < kl)[:, None, None], t[b], 0.0) for t in (k, v)]
        seen = visible(ql, kl, lq, lk, left, right)
        some = seen.any(1)
        for h in range(heads):
            x = torch.where((torch.arange(lq) < ql)[:, None], q[b, :, h], 0.0)
            y, z = keys[0][:, h // group], keys[1][:, h // group]
            s = torch.where(seen, scale * (x @ y.T), -math.inf)
            lse = torch.logsumexp(s, 1) if lk else torch.full((lq,), -math.inf, dtype=torch.float64)
            p = torch.where(seen, torch.exp(s - torch.where(some, lse, 0.0)[:, None]), 0.0)
            o = p @ z
            want['out'][b, :, h], want['lse'][b, h] = o, lse
            # a score is off by its products' roundings, a probability by its score's,
            # its reference's and the exponential's (and its argument's own rounding)
            size = scale * (x.abs() @ y.abs().T)
            ds = (dim + 4) * E * size.amax() if size.numel() else torch.tensor(0.0)
            top = torch.where(seen, s.abs(), 0.0).amax() if s.numel() else torch.tensor(0.0)
            ep = 2 * ds + 8 * E * (1 + top) + (lk + 8) * E
            absolute = p @ z.abs()
            mass = seen.double() @ z.abs()
            far['out'][b, :, h] = (2 * u + ep + (lk + 8) * E) * absolute + tiny * (mass + 1)
            far['lse'][b, h] = torch.where(some, ds + (lk + 16) * E * (1 + lse.abs()), 0.0)
            if dout is None:
                continue
            g = torch.where((torch.arange(lq) < ql)[:, None], do[b, :, h], 0.0)
            dp = g @ z.T
            delta = (g * o).sum(1, keepdim=True)
            dscore = p * (dp - delta)
            out_off = far['out'][b, :, h] + u * o.abs()
            off = (p * ((dim + 4) * E * (g.abs() @ z.abs().T) + (dim + 4) * E * (g.abs() * o.abs()).sum(1, keepdim=True)
                        + (g.abs() * out_off).sum(1, keepdim=True))
                   + (u + 2 * ep) * dscore.abs() + torch.where(seen, tiny + LEAST * (dp - delta).abs(), 0.0))
            want['dq'][b, :, h] = scale * (dscore @ y)
            want['dk'][b, :, h // group] += scale * (dscore.T @ x)
            want['dv'][b, :, h // group] += p.T @ g
            n = (lk + lq * group + 8) * E
            far['dq'][b, :, h] = scale * ((off + n * dscore.abs()) @ y.abs()) + u * want['dq'][b, :, h].abs() + tiny
            far['dk'][b, :, h // group] += scale * ((off + n * dscore.abs()).T @ x.abs())
            far['dv'][b, :, h // group] += ((u + 2 * ep + n) * p + torch.where(seen, tiny, 0.0)).T @ g.abs()
    if dout is not None:
        for n in ('dk', 'dv'):
            far[n] += u * want[n].abs() + tiny
    return {n: (want[n], far[n]) for n in names}


def check(got, want, far, name):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, name
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~(off <= far)
    assert not bad.any(), (name, int(bad.sum()), float(off.nan_to_num(math.inf).max()),
                           float((off / far.clamp(min=1e-300)).nan_to_num(math.inf).max()))


def philox(counter, seed):
    """Words (n, 4) of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, 2011) at uint64 counters."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    counter = np.asarray(counter, np.uint64)
    x = [counter & low, counter >> half, np.zeros_like(counter), np.zeros_like(counter)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> half) ^ x[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ x[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(x, -1)


def keep(rows, columns, probability, seed, offset=0):
    """(rows, columns) bool: the elements that dropout keeps."""
    count = rows * columns
    with np.errstate(over='ignore'):
        counter = np.uint64(offset) + np.arange((count + 3) // 4, dtype=np.uint64)
    words = philox(counter, seed).reshape(-1)[:count].reshape(rows, columns)
    return torch.from_numpy(words >= np.uint64(round(probability * 2 ** 32)))
