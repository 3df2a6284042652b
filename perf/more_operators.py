"""More of the sequence operators by which this framework is measured: what a layer
computes around its attention, and how its matrices are updated.

A case is one call, or one forward and its gradient, as a program that uses the
framework makes it on inputs made from a seed:

  * ``linear``        act(x W^T + bias) + residual;
  * ``linear_train``  the same, then the gradients of x, W and bias;
  * ``rotate``        queries and keys of one layer: each head's norm, then its rotation
                      by the token's position;
  * ``rotate_train``  the same, then the gradients of queries, keys and both norms' weights;
  * ``orthogonal``    matrices brought near the orthogonal ones of their singular vectors;
  * ``update``        one step of weights along such a matrix, made from the momentum.

The plain forms below compute in 32 bits with elementary torch operations (angles and
the sum under a matrix's norm in 64).
"""
import math
import random

import torch

own = False

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
ACTIVATIONS = ('none', 'sigmoid', 'relu', 'silu', 'gelu')
BASE, EPS = 10000.0, 1e-6
QUINTIC, STEPS = (3.4445, -4.7750, 2.0315), 5     # of the products that orthogonalise
RATE, DECAY, MOMENTUM = 0.02, 0.1, 0.95


def _linear(name, call, dtype, rows, inputs, outputs, activation, bias=True, residual=False):
    return {'name': name, 'call': call, 'dtype': dtype, 'rows': rows, 'inputs': inputs, 'outputs': outputs,
            'activation': activation, 'bias': bias, 'residual': residual}


def _rotation(name, call, dtype, batch, tokens, heads, kv_heads, dim, rotated, interleaved=False, far=False, ragged=False):
    return {'name': name, 'call': call, 'dtype': dtype, 'batch': batch, 'tokens': tokens, 'heads': heads,
            'kv_heads': kv_heads, 'dim': dim, 'rotated': rotated, 'interleaved': interleaved, 'far': far, 'ragged': ragged}


def _matrices(name, call, dtype, count, rows, columns):
    return {'name': name, 'call': call, 'dtype': dtype, 'count': count, 'rows': rows, 'columns': columns}


def listed():
    return [
        # a layer's wide product for single tokens of 16 sequences: the weights are read once
        _linear('linear_token', 'linear', 'bf16', 16, 2048, 8192, 'silu', bias=False),
        # four of the published grid's point sets through a layer of the published width,
        # in the framework's own precision: latency is much of it
        _linear('linear_points', 'linear', 'f32', 2916, 128, 128, 'sigmoid', residual=True),
        # a long prompt through a layer's wide product: matrix products are all of it
        _linear('linear_long', 'linear', 'bf16', 16384, 2048, 8192, 'gelu'),
        # eight point sets of the published grid in training
        _linear('linear_train_points', 'linear_train', 'f32', 5832, 128, 512, 'sigmoid'),
        # a training step's tokens through a layer
        _linear('linear_train', 'linear_train', 'bf16', 8192, 2048, 4096, 'gelu', residual=True),
        # single tokens of 16 sequences, far along
        _rotation('rotate_token', 'rotate', 'bf16', 16, 1, 16, 4, 128, 128, far=True),
        # point sets of the published grid in training
        _rotation('rotate_train_points', 'rotate_train', 'f32', 4, 729, 4, 4, 32, 32),
        # long sequences in training, some shorter than the others: memory is all of it
        _rotation('rotate_train', 'rotate_train', 'bf16', 2, 8192, 16, 4, 128, 128, ragged=True),
        # the hidden layers of the published network
        _matrices('orthogonal_layers', 'orthogonal', 'f32', 4, 128, 128),
        # tall matrices, no size round
        _matrices('orthogonal_odd', 'orthogonal', 'f16', 2, 1000, 333),
        # the wide product's matrix of a layer
        _matrices('orthogonal', 'orthogonal', 'bf16', 1, 2048, 8192),
        # the four square matrices of a layer in training, in the framework's own precision
        _matrices('update', 'update', 'f32', 4, 1024, 1024),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A width: mostly whole eights."""
    n = _spread(rng, low, high)
    return max(8, n // 8 * 8) if rng.random() < 0.75 else n


def draw(rng: random.Random):
    call = rng.choice(['linear', 'linear', 'token', 'linear_train', 'linear_train', 'rotate', 'rotate_train', 'orthogonal',
                       'update'])
    dtype = rng.choice(['f32', 'f16', 'bf16', 'bf16'])
    if call in ('linear', 'token', 'linear_train'):
        c = _linear('', 'linear' if call == 'token' else call, dtype, rng.randint(1, 48) if call == 'token' else _spread(rng, 16, 16384),
                    _width(rng, 8, 8192), _width(rng, 8, 8192), rng.choice(ACTIVATIONS), rng.random() < 0.6, rng.random() < 0.4)
        while work(c)['flops'] > (5e10 if dtype == 'f32' else 5e11):
            k = max(('rows', 'inputs', 'outputs'), key=lambda k: c[k])
            c[k] //= 2
    elif call in ('rotate', 'rotate_train'):
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 5])
        dim = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128])
        c = _rotation('', call, dtype, rng.randint(1, 16), rng.randint(1, 3) if rng.random() < 0.3 else _spread(rng, 4, 8192),
                      heads, kv_heads, dim, rng.choice([dim, dim, dim // 2, dim // 4 * 2]), rng.random() < 0.4,
                      rng.random() < 0.4, rng.random() < 0.4)
        while c['batch'] * c['tokens'] * (heads + kv_heads) * dim > 2 * 8192 * 20 * 128:
            if c['batch'] > 1:
                c['batch'] //= 2
            else:
                c['tokens'] //= 2
    else:
        c = _matrices('', call, dtype, rng.choice([1, 1, 2, 4, 6]), _width(rng, 8, 4096), _width(rng, 8, 4096))
        while work(c)['flops'] > (3e10 if dtype == 'f32' else 3e11):
            if c['count'] > 1:
                c['count'] //= 2
            else:
                k = max(('rows', 'columns'), key=lambda k: c[k])
                c[k] //= 2
    del c['name']
    return c


def work(case):
    size, call = TYPES[case['dtype']].itemsize, case['call']
    if call in ('linear', 'linear_train'):
        n, i, o = case['rows'], case['inputs'], case['outputs']
        values = n * i + i * o + n * o * (1 + case['residual']) + o * case['bias']
        if call == 'linear':
            return {'bytes': size * values, 'flops': 2.0 * n * i * o}
        # dy in; dx, dW, dbias out; three products
        return {'bytes': size * (values + n * o + n * i + i * o + o * case['bias']), 'flops': 6.0 * n * i * o}
    if call in ('rotate', 'rotate_train'):
        values = case['batch'] * case['tokens'] * (case['heads'] + case['kv_heads']) * case['dim']
        passes = 2 if call == 'rotate' else 4     # x, y, dy, dx
        return {'bytes': size * (passes * values + passes * case['dim']) + 4 * case['batch'] * case['tokens'],
                'flops': (7.0 if call == 'rotate' else 22.0) * values}
    n = case['count'] * case['rows'] * case['columns']
    r, c = sorted((case['rows'], case['columns']))
    # a step's two symmetric products, by halves, and a whole one
    flops = float(case['count'] * STEPS * (r * r * c + r * r * r + 2 * r * r * c))
    if call == 'orthogonal':
        return {'bytes': size * 2 * n, 'flops': flops}
    # the gradient in, weights and (32-bit) momentum in and out
    return {'bytes': (3 * size + 8) * n, 'flops': flops}


# ----------------------------------------------------------------------------- inputs
_device = None


def _library():
    """The framework's binding, and its device on torch's stream."""
    global _device
    from cpde_amd import hip
    if _device is None:
        _device = hip.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    return hip, _device


def _inputs(case, seed):
    """Tensors of a case: activations as a layer hands them on (normal), gradients of a mean's size."""
    g = torch.Generator('cuda').manual_seed(seed)
    dtype = TYPES[case['dtype']]

    def normal(*shape, scale=1.0, type_=dtype):
        return torch.empty(shape, device='cuda', dtype=type_).normal_(0, scale, generator=g)

    s = {'case': dict(case)}
    if case['call'] in ('linear', 'linear_train'):
        n, i, o = case['rows'], case['inputs'], case['outputs']
        s['x'], s['weight'] = normal(n, i), normal(o, i, scale=i ** -0.5)
        if case['bias']:
            s['bias'] = normal(o, scale=0.1)
        if case['residual']:
            s['residual'] = normal(n, o)
        if case['call'] == 'linear_train':
            s['dy'] = normal(n, o, scale=0.1)
    elif case['call'] in ('rotate', 'rotate_train'):
        b, t, h, hk, d = (case[k] for k in ('batch', 'tokens', 'heads', 'kv_heads', 'dim'))
        s['q'], s['k'] = normal(b, t, h, d, scale=2.0), normal(b, t, hk, d)
        s['q_weight'], s['k_weight'] = 1 + normal(d, scale=0.2), 1 + normal(d, scale=0.2)
        first = torch.randint(0, (1 << 20) if case['far'] else 1, (b, 1), device='cuda', generator=g)
        at = torch.arange(t, device='cuda')[None] + first
        if case['ragged']:
            # every entry ends somewhere else, the last at its full length
            ends = torch.tensor([t * (i + 1) // b for i in range(b)], device='cuda')[:, None]
            at = torch.where(torch.arange(t, device='cuda')[None] < ends, at, -1)
        s['positions'] = at.int()
        if case['call'] == 'rotate_train':
            s['dq_out'], s['dk_out'] = normal(b, t, h, d, scale=0.1), normal(b, t, hk, d, scale=0.1)
    else:
        n, r, c = case['count'], case['rows'], case['columns']
        # a gradient: noise, and a few directions that stand out of it
        common = torch.matmul(normal(n, r, 4, type_=torch.float32), normal(n, 4, c, type_=torch.float32))
        gradient = ((normal(n, r, c, type_=torch.float32) + common) * 1e-3).to(dtype)
        if case['call'] == 'orthogonal':
            s['x'] = gradient
        else:
            s['gradient'] = gradient
            s['momentum'] = normal(n, r, c, scale=4e-3, type_=torch.float32)
            s['weight'] = normal(n, r, c, scale=c ** -0.5)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    hip, device = _library()
    dtype = {'f32': hip.F32, 'f16': hip.F16, 'bf16': hip.BF16}[case['dtype']]
    train = case['call'].endswith('_train')
    views = s['views'] = {}
    if case['call'] in ('linear', 'linear_train'):
        activation = {'none': hip.NONE, 'sigmoid': hip.SIGMOID, 'relu': hip.RELU, 'silu': hip.SILU, 'gelu': hip.GELU}
        s['plan'] = hip.Linear(device, dtype, case['rows'], case['inputs'], case['outputs'], activation[case['activation']],
                               backward=train)
        s['y'] = torch.empty((case['rows'], case['outputs']), device='cuda', dtype=TYPES[case['dtype']])
        if train:
            s['dx'], s['dweight'] = torch.empty_like(s['x']), torch.empty_like(s['weight'])
            if case['bias']:
                s['dbias'] = torch.empty_like(s['bias'])
            if case['activation'] != 'none':
                s['pre'] = torch.empty_like(s['y'])
        for k in ('x', 'weight', 'residual', 'y', 'pre', 'dy', 'dx', 'dweight'):
            if k in s:
                views[k] = hip.Rows.of(s[k])
    elif case['call'] in ('rotate', 'rotate_train'):
        s['plan'] = hip.Rotation(device, dtype, case['batch'], case['tokens'], case['heads'], case['kv_heads'], case['dim'],
                                 rotated=case['rotated'], interleaved=case['interleaved'], base=BASE, eps=EPS, backward=train)
        s['q_out'], s['k_out'] = torch.empty_like(s['q']), torch.empty_like(s['k'])
        if train:
            s['dq'], s['dk'] = torch.empty_like(s['q']), torch.empty_like(s['k'])
            s['dq_weight'], s['dk_weight'] = torch.empty_like(s['q_weight']), torch.empty_like(s['k_weight'])
        for k in ('q', 'k', 'q_out', 'k_out', 'dq_out', 'dk_out', 'dq', 'dk'):
            if k in s:
                views[k] = hip.Heads.of(s[k])
    else:
        s['plan'] = hip.Orthogonal(device, dtype, case['count'], case['rows'], case['columns'], steps=STEPS)
        if case['call'] == 'orthogonal':
            s['out'] = torch.empty_like(s['x'])
        for k in ('x', 'out', 'gradient', 'momentum', 'weight'):
            if k in s:
                views[k] = hip.Matrices.of(s[k])
    return s


# ----------------------------------------------------------------------------- the plain forms
def _plain_linear(s):
    c, dtype = s['case'], s['x'].dtype
    x, weight = s['x'].float(), s['weight'].float()
    z = torch.matmul(x, weight.t())
    if c['bias']:
        z += s['bias'].float()
    act = c['activation']
    if act in ('sigmoid', 'silu'):
        gate = torch.sigmoid(z)
    elif act == 'gelu':
        gate = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    y = {'none': lambda: z, 'sigmoid': lambda: gate, 'relu': lambda: z.clamp(min=0), 'silu': lambda: z * gate,
         'gelu': lambda: z * gate}[act]()
    if c['residual']:
        y = y + s['residual'].float()
    result = {'y': y.to(dtype)}
    del y
    if c['call'] == 'linear':
        return result
    slope = {'none': lambda: 1.0, 'sigmoid': lambda: gate * (1 - gate), 'relu': lambda: (z > 0).float(),
             'silu': lambda: gate * (1 + z * (1 - gate)),
             'gelu': lambda: gate + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))}[act]()
    dz = s['dy'].float() * slope
    result['dx'] = torch.matmul(dz, weight).to(dtype)
    result['dweight'] = torch.matmul(dz.t(), x).to(dtype)
    if c['bias']:
        result['dbias'] = dz.sum(0).to(dtype)
    return result


def _angles(s):
    """cos and sin [batch, tokens, 1, rotated / 2] in 32 bits, of angles in 64; and which tokens there are."""
    c, at = s['case'], s['positions'].double()
    rate = BASE ** (-torch.arange(0, c['rotated'], 2, device='cuda', dtype=torch.float64) / max(1, c['rotated']))
    angle = (at[..., None] * rate)[:, :, None]
    return torch.cos(angle).float(), torch.sin(angle).float(), (at >= 0)[:, :, None, None]


def _split(c, x):
    """The two halves of the rotated pairs, and the rest."""
    n = c['rotated']
    if c['interleaved']:
        return x[..., 0:n:2], x[..., 1:n:2], x[..., n:]
    return x[..., :n // 2], x[..., n // 2:n], x[..., n:]


def _joined(c, a, b, rest):
    pairs = torch.stack([a, b], -1).flatten(-2) if c['interleaved'] else torch.cat([a, b], -1)
    return torch.cat([pairs, rest], -1)


def _plain_rotation(s):
    c = s['case']
    cos, sin, there = _angles(s)
    result = {}
    for n in ('q', 'k'):
        x, weight = s[n].float(), s[n + '_weight'].float()
        up = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        normed = x * up
        a, b, rest = _split(c, normed * weight)
        y = _joined(c, a * cos - b * sin, a * sin + b * cos, rest)
        result[n + '_out'] = torch.where(there, y, 0.0).to(s[n].dtype)
        if c['call'] == 'rotate_train':
            a, b, rest = _split(c, torch.where(there, s[f'd{n}_out'].float(), 0.0))
            dy = _joined(c, a * cos + b * sin, b * cos - a * sin, rest)
            result[f'd{n}_weight'] = (dy * normed).flatten(0, 2).sum(0).to(s[n].dtype)
            dy = dy * weight
            dx = up * (dy - normed * (dy * normed).mean(-1, keepdim=True))
            result['d' + n] = torch.where(there, dx, 0.0).to(s[n].dtype)
    return result


def _plain_orthogonal(x):
    """Near U V^T of x = U S V^T, by products; x in 32 bits, [count, rows, columns]."""
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    norm = x.double().square().sum((1, 2), keepdim=True).sqrt()
    x = x * torch.where(norm > 0, 1 / norm, 0.0).float()
    a, b, c = QUINTIC
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(1, 2) if tall else x


def _plain_update(s):
    c, dtype = s['case'], s['weight'].dtype
    gradient = s['gradient'].float()
    s['momentum'].mul_(MOMENTUM).add_(gradient)
    step = _plain_orthogonal(gradient + MOMENTUM * s['momentum'])
    size = RATE * math.sqrt(max(1.0, c['rows'] / c['columns']))
    s['weight'].copy_((s['weight'].float() * (1 - RATE * DECAY) - size * step).to(dtype))
    return {'momentum': s['momentum'], 'weight': s['weight']}


# ----------------------------------------------------------------------------- the calls
def run(s):
    c = s['case']
    if not own:
        if c['call'] in ('linear', 'linear_train'):
            return _plain_linear(s)
        if c['call'] in ('rotate', 'rotate_train'):
            return _plain_rotation(s)
        if c['call'] == 'update':
            return _plain_update(s)
        return {'out': _plain_orthogonal(s['x'].float()).to(s['x'].dtype)}
    w, plan = s['views'], s['plan']
    if c['call'] in ('linear', 'linear_train'):
        plan.forward(c['rows'], w['x'], w['weight'], w['y'], bias=s.get('bias'), residual=w.get('residual'), pre=w.get('pre'))
        result = {'y': s['y']}
        if c['call'] == 'linear_train':
            plan.backward(c['rows'], w['x'], w['weight'], w['dy'], pre=w.get('pre'), dx=w['dx'], dweight=w['dweight'],
                          dbias=s.get('dbias'))
            result.update({k: s[k] for k in ('dx', 'dweight', 'dbias') if k in s})
        return result
    if c['call'] in ('rotate', 'rotate_train'):
        plan.forward(w['q'], w['k'], w['q_out'], w['k_out'], s['q_weight'], s['k_weight'], s['positions'])
        result = {'q_out': s['q_out'], 'k_out': s['k_out']}
        if c['call'] == 'rotate_train':
            plan.backward(w['q'], w['k'], w['dq_out'], w['dk_out'], w['dq'], w['dk'], s['q_weight'], s['k_weight'],
                          s['dq_weight'], s['dk_weight'], s['positions'])
            result.update({k: s[k] for k in ('dq', 'dk', 'dq_weight', 'dk_weight')})
        return result
    if c['call'] == 'orthogonal':
        plan.forward(w['x'], w['out'])
        return {'out': s['out']}
    plan.update(w['gradient'], w['momentum'], w['weight'], rate=RATE, momentum_factor=MOMENTUM, decay=DECAY, nesterov=True)
    return {'momentum': s['momentum'], 'weight': s['weight']}


# ----------------------------------------------------------------------------- 64 bits
def _exact_linear(s):
    """The gradients by automatic differentiation."""
    c = s['case']
    names = [n for n in ('x', 'weight', 'bias') if n in s]
    leaf = {n: s[n].double().requires_grad_(c['call'] == 'linear_train') for n in names}
    z = torch.nn.functional.linear(leaf['x'], leaf['weight'], leaf.get('bias'))
    y = {'none': lambda t: t, 'sigmoid': torch.sigmoid, 'relu': torch.relu, 'silu': torch.nn.functional.silu,
         'gelu': torch.nn.functional.gelu}[c['activation']](z)
    if c['residual']:
        y = y + s['residual']
    result = {'y': y.detach()}
    if c['call'] == 'linear_train':
        grads = torch.autograd.grad(y, list(leaf.values()), s['dy'].double())
        result.update({'d' + n: g for n, g in zip(names, grads)})
    return result


def _exact_rotation(s):
    """Pairs as complex numbers, turned by complex factors; the gradients by automatic differentiation."""
    c = s['case']
    at = s['positions'].double()
    n = c['rotated']
    turn = torch.exp(1j * at[:, :, None, None] * BASE ** (-torch.arange(n // 2, device='cuda', dtype=torch.float64) * 2 / max(1, n)))
    result = {}
    for name in ('q', 'k'):
        train = c['call'] == 'rotate_train'
        x, weight = (s[k].double().requires_grad_(train) for k in (name, name + '_weight'))
        scaled = x / torch.sqrt(torch.mean(x ** 2, -1, keepdim=True) + EPS) * weight
        head = scaled[..., :n].unflatten(-1, (-1, 2) if c['interleaved'] else (2, -1))
        if not c['interleaved']:
            head = head.transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn)
        if not c['interleaved']:
            turned = turned.transpose(-1, -2)
        y = torch.cat([turned.flatten(-2), scaled[..., n:]], -1) * (at >= 0)[:, :, None, None]
        result[name + '_out'] = y.detach()
        if train:
            result['d' + name], result[f'd{name}_weight'] = torch.autograd.grad(y, (x, weight), s[f'd{name}_out'].double())
    return result


def _exact_orthogonal(x):
    """The same polynomial of the singular values, one matrix at a time."""
    out = torch.zeros_like(x)
    for i, m in enumerate(x):
        norm = torch.linalg.matrix_norm(m)
        if norm == 0:
            continue
        m = m / norm
        for _ in range(STEPS):
            if m.shape[0] <= m.shape[1]:
                gram = torch.matmul(m, m.t())
                inner = torch.matmul(gram, m)
                m = QUINTIC[0] * m + QUINTIC[1] * inner + QUINTIC[2] * torch.matmul(gram, inner)
            else:
                gram = torch.matmul(m.t(), m)
                inner = torch.matmul(m, gram)
                m = QUINTIC[0] * m + QUINTIC[1] * inner + QUINTIC[2] * torch.matmul(inner, gram)
        out[i] = m
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case['call'] in ('linear', 'linear_train'):
        return _exact_linear(s)
    if case['call'] in ('rotate', 'rotate_train'):
        return _exact_rotation(s)
    if case['call'] == 'orthogonal':
        return {'out': _exact_orthogonal(s['x'].double())}
    momentum = MOMENTUM * s['momentum'].double() + s['gradient']
    step = _exact_orthogonal(s['gradient'] + MOMENTUM * momentum)
    size = RATE * max(1.0, case['rows'] / case['columns']) ** 0.5
    return {'momentum': momentum, 'weight': (1 - RATE * DECAY) * s['weight'].double() - size * step}
