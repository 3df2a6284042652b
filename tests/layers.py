"""The layer operators (products with epilogues, head rotations, orthogonal updates) in
float64, with bounds on how far a kernel's results may lie from them.

Bounds are worst cases of the kernels' own steps, first order, element by element: u is
half a unit in the last place of the tensors' type, E = 2^-24 that of float sums (a sum of
n products is off by at most n + 8 of them), tiny where roundings become absolute."""
import math

import torch

from sequences import E, TINY, UNIT

ACTIVATIONS = ['none', 'sigmoid', 'relu', 'silu', 'gelu']
PAIR = 2.0 ** -22      # a sum of two f16 values
QUINTIC = (3.4445, -4.7750, 2.0315)


def activation(kind, z):
    """Value and slope."""
    if kind == 'sigmoid':
        s = torch.sigmoid(z)
        return s, s * (1 - s)
    if kind == 'relu':
        return z.clamp(min=0), (z > 0).double()
    if kind == 'silu':
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if kind == 'gelu':
        s = torch.special.ndtr(z)
        return z * s, s + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def linear(x, weight, bias, residual, kind, dtype):
    """{name: (values, bounds)} of y and pre."""
    u, tiny = UNIT[dtype], TINY[dtype]
    x, weight = x.double(), weight.double()
    z = x @ weight.T
    # six products of split floats, or one
    size = x.abs() @ weight.abs().T
    off = (6 * x.shape[1] + 16) * E * size
    if bias is not None:
        z = z + bias.double()
        off = off + E * z.abs()
    y, _ = activation(kind, z)
    # no slope passes 1.13; values are off by a few units of float besides
    y_off = 1.13 * off + (0 if kind == 'none' else 16 * E * (1 + z.abs()))
    if residual is not None:
        y = y + residual.double()
        y_off = y_off + E * y.abs()
    return {'y': (y, y_off + u * (y.abs() + y_off) + tiny), 'pre': (z, off + u * (z.abs() + off) + tiny)}


def linear_gradient(x, weight, pre, dy, kind, dtype, before=None):
    """{name: (values, bounds)} of dx, dweight and dbias; before: what dweight and dbias are added onto."""
    u, tiny = UNIT[dtype], TINY[dtype]
    x, weight, dy = x.double(), weight.double(), dy.double()
    dz, off = dy, torch.zeros_like(dy)
    if kind != 'none':
        dz = dy * activation(kind, pre.double())[1]
        off = u * dz.abs() + 16 * E * (1 + pre.double().abs()) * dy.abs() + tiny
    rows, outputs = dz.shape
    result = {'dx': (dz @ weight, off @ weight.abs() + (6 * outputs + 16) * E * (dz.abs() @ weight.abs())),
              'dweight': (dz.T @ x, off.T @ x.abs() + (6 * rows + 16) * E * (dz.abs().T @ x.abs())),
              'dbias': (dz.sum(0), off.sum(0) + (rows + 16) * E * dz.abs().sum(0))}
    for n, b in (before or {}).items():
        result[n] = (result[n][0] + b.double(), result[n][1] + E * b.double().abs())
    return {n: (v, o + u * (v.abs() + o) + tiny) for n, (v, o) in result.items()}


def _pairs(x, rotated, interleaved):
    if interleaved:
        return x[..., 0:rotated:2], x[..., 1:rotated:2], x[..., rotated:]
    return x[..., :rotated // 2], x[..., rotated // 2:rotated], x[..., rotated:]


def _unpairs(a, b, rest, interleaved):
    pairs = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([pairs, rest], -1)


def rotation(x, weight, positions, rotated, interleaved, base, eps, norm, dtype, dy=None):
    """{name: (values, bounds)} of out and, with dy, dx and dweight; x [batch][token][head][dim]."""
    u, tiny = UNIT[dtype], TINY[dtype]
    dim = x.shape[-1]
    there = (positions >= 0)[:, :, None, None]
    x = torch.where(there, x.double(), 0.0)
    w = torch.ones(dim, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    rate = base ** (-2 * torch.arange(rotated // 2, dtype=torch.float64, device=x.device) / max(1, rotated))
    angle = (positions.double()[..., None] * rate)[:, :, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    # sines off by 8 units of float, and by the roundings of far angles in double on both sides
    turn_off = 8 * E + 8 * 2.0 ** -52 * angle.abs()
    up = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) if norm else torch.ones_like(x[..., :1])
    normed = x * up
    a, b, rest = _pairs(normed * w, rotated, interleaved)
    y = _unpairs(a * cos - b * sin, a * sin + b * cos, rest, interleaved)
    both = a.abs() + b.abs()
    far = (dim + 32) * E
    y_off = _unpairs(both * (far + turn_off), both * (far + turn_off), rest.abs() * far, interleaved)
    result = {'out': (torch.where(there, y, 0.0), torch.where(there, y_off + u * (y.abs() + y_off) + tiny, 0.0))}
    if dy is None:
        return result
    ga, gb, rest = _pairs(torch.where(there, dy.double(), 0.0), rotated, interleaved)
    g = _unpairs(ga * cos + gb * sin, gb * cos - ga * sin, rest, interleaved)
    both = ga.abs() + gb.abs()
    g_off = _unpairs(both * (8 * E + turn_off), both * (8 * E + turn_off), rest.abs() * 8 * E, interleaved)
    size = g.abs() + g_off
    rows = x[..., 0].numel()
    dw = (g * normed).flatten(0, 2).sum(0)
    dw_off = ((g_off + (rows + dim + 32) * E * size) * normed.abs()).flatten(0, 2).sum(0)
    gw = g * w
    mean = (gw * normed).mean(-1, keepdim=True) if norm else 0.0
    dx = up * (gw - normed * mean)
    gw_size = size * w.abs()
    spread = normed.abs() * (gw_size * normed.abs()).mean(-1, keepdim=True) if norm else 0.0
    spread_off = normed.abs() * (g_off * w.abs() * normed.abs()).mean(-1, keepdim=True) if norm else 0.0
    dx_off = up * (g_off * w.abs() + spread_off + (3 * dim + 64) * E * (gw_size + spread))
    result['dx'] = (torch.where(there, dx, 0.0), torch.where(there, dx_off + u * (dx.abs() + dx_off) + tiny, 0.0))
    result['dweight'] = (dw, dw_off + u * (dw.abs() + dw_off) + tiny)
    return result


def orthogonal(x, steps):
    """O(x) of matrices [count][rows][columns], on the smaller side."""
    tall = x.shape[1] > x.shape[2]
    x = x.double()
    x = x.transpose(1, 2) if tall else x
    norm = x.square().sum((1, 2), keepdim=True).sqrt()
    x = torch.where(norm > 0, x / norm, 0.0)
    a, b, c = QUINTIC
    for _ in range(steps):
        gram = x @ x.transpose(1, 2).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.transpose(1, 2) if tall else x).contiguous()


def orthogonal_first(x, dtype):
    """(values, bounds) of one step.  Operands of the products are off by half a unit of f16
    (bf16 matrices) or of a sum of two of them; in the first case without the diagonals of A and
    of b A + c A^2, which stay as they are."""
    a, b, c = QUINTIC
    h = 2.0 ** -11 if dtype == 'bf16' else PAIR
    least = 2.0 ** -24 / 4096      # of an operand times 2^12
    tall = x.shape[1] > x.shape[2]
    x = x.double()
    x = x.transpose(1, 2) if tall else x
    norm = x.square().sum((1, 2), keepdim=True).sqrt()
    x = torch.where(norm > 0, x / norm, 0.0)
    r, k = x.shape[1:]
    size = x.abs() @ x.abs().transpose(1, 2).contiguous()
    gram = x @ x.transpose(1, 2).contiguous()
    spread = x.abs().sum(2)
    gram_off = (2 * h + (3 * k + 16) * E) * size + least * (spread[:, :, None] + spread[:, None, :])
    off = torch.ones_like(gram[0]) - (torch.eye(r, dtype=torch.float64, device=x.device) if dtype == 'bf16' else 0)
    gram_off = gram_off + off * (h * (gram.abs() + gram_off) + least)
    inner = gram.abs() + gram_off
    square_off = inner @ gram_off + gram_off @ inner + (3 * r + 16) * E * (inner @ inner)
    poly = b * gram + c * (gram @ gram)
    poly_off = abs(b) * gram_off + c * square_off + 8 * E * (1 + gram.abs())
    poly_off = poly_off + off * (h * (poly.abs() + poly_off) + least)
    y = a * x + poly @ x
    # (X itself is a sum of two f16 values, to `least` where it is small; in products one)
    y_off = (a * (PAIR * x.abs() + least) + ((1 - off) * poly.abs()) @ (PAIR * x.abs() + least) + poly_off @ x.abs()
             + (off * (poly.abs() + poly_off)) @ (h * x.abs() + least)
             + (3 * r + 16) * E * (poly.abs() @ x.abs()) + 8 * E * (a * x.abs() + y.abs()))
    y_off = y_off + UNIT[dtype] * (y.abs() + y_off) + TINY[dtype]
    return tuple((t.transpose(1, 2) if tall else t).contiguous() for t in (y, y_off))


def orthogonal_far(dtype, inner):
    """How far (2-norm over 2-norm) five steps may be off.  A step's sum a X + b A X + c A^2 X
    has absolute weights of at most 3.44 + 4.78 * 1.44 + 2.03 * 2.07 = 14.5 on matrices whose
    largest singular value is 1.2; its roundings are independent: of the operands (five, rms
    half of their bound) and of sums over `inner` terms (rms a half unit for the root of
    their number, three products)."""
    h = 2.0 ** -11 if dtype == 'bf16' else PAIR
    return 14.5 * math.sqrt(25) * (h / 2 + math.sqrt(3 * inner) * E / 2) + UNIT[dtype]
