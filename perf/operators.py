"""The sequence operators by which this framework is measured: attention and its
gradient, the embedding lookup and its gradient, dropout.

A case is one call, or one forward and its gradient, as a program that uses the
framework makes it on inputs made from a seed:

  * ``attend``   attention forward;
  * ``train``    attention forward, then its gradient;
  * ``lookup``   rows of an embedding table, scaled;
  * ``scatter``  the gradient of that table;
  * ``dropout``  dropout of one tensor added onto another, and its gradient.

The plain forms below compute in 32 bits with elementary torch operations.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
ROUND_KEYS, MULTIPLIERS = (0x9E3779B9, 0xBB67AE85), (0xD2511F53, 0xCD9E8D57)  # Philox4x32
OFFSET = 1 << 33  # of the generator's counter: past 32 bits, as in a long training run


def _attention(name, call, dtype, batch, queries, keys, heads, kv_heads, dim, left=-1, right=-1, ragged=False):
    return {'name': name, 'call': call, 'dtype': dtype, 'batch': batch, 'queries': queries, 'keys': keys, 'heads': heads,
            'kv_heads': kv_heads, 'dim': dim, 'left': left, 'right': right, 'ragged': ragged}


def _embedding(name, call, dtype, tokens, rows, width, skewed, wide_ids=False):
    return {'name': name, 'call': call, 'dtype': dtype, 'tokens': tokens, 'rows': rows, 'width': width,
            'skewed': skewed, 'wide_ids': wide_ids}


def _dropout(name, dtype, rows, width, probability):
    return {'name': name, 'call': 'dropout', 'dtype': dtype, 'rows': rows, 'width': width, 'probability': probability}


def listed():
    return [
        # one query against the 729 points of the published grid, in the
        # framework's own precision: latency is all of it
        _attention('step_points', 'attend', 'f32', 1, 1, 729, 4, 4, 32),
        # single tokens of 16 sequences against caches of all lengths
        _attention('step_cache', 'attend', 'bf16', 16, 1, 32768, 16, 4, 128, ragged=True),
        # point sets of the published grid attending to themselves
        _attention('points', 'attend', 'f32', 4, 729, 729, 4, 4, 32),
        # a long causal sequence with shared key heads: matrix products are all of it
        _attention('causal_long', 'attend', 'bf16', 2, 8192, 8192, 16, 4, 128, right=0),
        # the published grid's point sets in training, in the framework's own precision
        _attention('train_points', 'train', 'f32', 8, 729, 729, 4, 4, 32),
        # sets of queries reading ragged sets of sensors, no size round
        _attention('train_cross', 'train', 'f16', 5, 1000, 333, 6, 2, 80, ragged=True),
        # causal training at the usual length
        _attention('train_causal', 'train', 'bf16', 2, 4096, 4096, 16, 4, 128, right=0),
        # a batch of tokens looked up in a large table
        _embedding('lookup', 'lookup', 'bf16', 32768, 65536, 1024, True),
        # the gradient of a small table: launches are most of it
        _embedding('scatter_small', 'scatter', 'f32', 2187, 1000, 128, False),
        # the gradient of a large table on tokens of very uneven frequency
        _embedding('scatter', 'scatter', 'bf16', 131072, 65536, 512, True, True),
        # the activations of one layer over the published grid
        _dropout('dropout_small', 'f32', 729, 128, 0.1),
        # and over the largest point set of the benchmark's configurations
        _dropout('dropout', 'bf16', 262144, 256, 0.1),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random):
    call = rng.choice(['attend', 'attend', 'step', 'train', 'train', 'lookup', 'scatter', 'scatter', 'dropout'])
    dtype = rng.choice(['f32', 'f16', 'bf16', 'bf16'])
    if call in ('attend', 'step', 'train'):
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 8])
        dim = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128])
        queries = rng.randint(1, 3) if call == 'step' else _spread(rng, 4, 8192)
        keys = _spread(rng, 16, 32768) if call == 'step' else queries if rng.random() < 0.6 else _spread(rng, 4, 8192)
        band = rng.random()
        left, right = (-1, 0) if band < 0.4 else (_spread(rng, 8, 1024), rng.choice([0, 64])) if band < 0.55 else (-1, -1)
        c = _attention('', 'attend' if call == 'step' else call, dtype, rng.randint(1, 16), queries, keys, heads, kv_heads,
                       dim, left, right, rng.random() < 0.3)
        # no more than the largest listed case; 32-bit products run at a sixteenth of the others' rate
        while (work(c)['flops'] * (16 if dtype == 'f32' else 1) > 5e11 or _pairs(c) * heads > 1.1e9
               or c['batch'] * c['keys'] * kv_heads * dim > 16 * 32768 * 4 * 128):
            if c['batch'] > 1:
                c['batch'] //= 2
            elif c['queries'] > c['keys']:
                c['queries'] //= 2
            else:
                c['keys'] //= 2
    elif call in ('lookup', 'scatter'):
        c = _embedding('', call, dtype, _spread(rng, 1, 131072), _spread(rng, 8, 65536), _spread(rng, 8, 1024),
                       rng.random() < 0.6, rng.random() < 0.5)
        if rng.random() < 0.8:
            c['width'] = max(8, c['width'] // 8 * 8)
        while c['tokens'] * c['width'] > 131072 * 512:
            c['tokens'] //= 2
        while c['rows'] * c['width'] > 65536 * 512:
            c['rows'] //= 2
    else:
        c = _dropout('', dtype, _spread(rng, 1, 262144), _spread(rng, 1, 1024), rng.choice([0.05, 0.1, 0.2, 0.5]))
        if rng.random() < 0.8:
            c['width'] = max(8, c['width'] // 8 * 8)
        while c['rows'] * c['width'] > 262144 * 128:
            c['rows'] //= 2
    del c['name']
    return c


# ----------------------------------------------------------------------------- sizes
def _lengths(case):
    """Tokens of each batch entry on both sides; a ragged batch spans all lengths and holds an empty one."""
    b = case['batch']
    if not case['ragged']:
        return [case['queries']] * b, [case['keys']] * b
    keys = [case['keys'] * (i + (b < 2)) // max(1, b - 1) for i in range(b)]
    queries = [case['queries'] if case['queries'] < 4 else max(1, case['queries'] * (b - i) // b) for i in range(b)]
    return queries, keys


def _pairs(case):
    """Visible (query, key) pairs of one head over the batch."""
    total = 0
    for ql, kl in zip(*_lengths(case)):
        if case['left'] < 0 and case['right'] < 0:
            total += ql * kl
            continue
        at = np.arange(ql) + kl - ql
        low = np.maximum(at - case['left'], 0) if case['left'] >= 0 else np.zeros(ql, np.int64)
        high = np.minimum(at + case['right'] + 1, kl) if case['right'] >= 0 else np.full(ql, kl)
        total += int(np.maximum(high - low, 0).sum())
    return total


def work(case):
    size = TYPES[case['dtype']].itemsize
    call = case['call']
    if call in ('attend', 'train'):
        ql, kl = _lengths(case)
        rows = case['batch'] * case['queries'] * case['heads'] * case['dim']      # outputs come whole
        read_rows = sum(ql) * case['heads'] * case['dim']
        read_keys = sum(kl) * case['kv_heads'] * case['dim']
        stats = 4 * case['batch'] * case['queries'] * case['heads']
        pairs = _pairs(case) * case['heads'] * case['dim']
        if call == 'attend':  # two products; q, k, v in; o and the logarithms of the sums out
            return {'bytes': size * (read_rows + 2 * read_keys + rows) + stats, 'flops': 4.0 * pairs}
        # and five more: the scores again, dp, dv, dk, dq; q, k, v, do in; o, the sums, dq, dk, dv out
        keys = case['batch'] * case['keys'] * case['kv_heads'] * case['dim']
        return {'bytes': size * (2 * read_rows + 2 * read_keys + 2 * rows + 2 * keys) + stats, 'flops': 14.0 * pairs}
    if call == 'lookup':
        # each row that occurs is read once: as many as the frequencies let expect
        at = np.arange(case['rows'] + 1) / case['rows']
        share = np.diff(at ** 0.25 if case['skewed'] else at)
        distinct = float((1 - (1 - share) ** case['tokens']).sum())
        return {'bytes': case['tokens'] * (8 if case['wide_ids'] else 4) + size * case['width'] * (distinct + case['tokens']),
                'flops': 1.0 * case['tokens'] * case['width']}
    if call == 'scatter':
        return {'bytes': case['tokens'] * (8 if case['wide_ids'] else 4) + size * case['width'] * case['tokens']
                + 4 * case['rows'] * case['width'], 'flops': 1.0 * case['tokens'] * case['width']}
    # x, the residual and dy in; y and dx out
    return {'bytes': 5 * size * case['rows'] * case['width'], 'flops': 3.0 * case['rows'] * case['width']}


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
    """Tensors of a case: activations as a layer hands them on (normal), gradients of a mean's size, token numbers."""
    g = torch.Generator('cuda').manual_seed(seed)
    dtype = TYPES[case['dtype']]

    def normal(*shape, scale=1.0):
        return torch.empty(shape, device='cuda', dtype=dtype).normal_(0, scale, generator=g)

    s = {'case': dict(case)}
    if case['call'] in ('attend', 'train'):
        b, lq, lk, h, hk, d = (case[k] for k in ('batch', 'queries', 'keys', 'heads', 'kv_heads', 'dim'))
        s['q'], s['k'], s['v'] = normal(b, lq, h, d), normal(b, lk, hk, d), normal(b, lk, hk, d)
        if case['call'] == 'train':
            s['dout'] = normal(b, lq, h, d, scale=0.1)
        if case['ragged']:
            ql, kl = _lengths(case)
            s['ql'] = torch.tensor(ql, dtype=torch.int32, device='cuda')
            s['kl'] = torch.tensor(kl, dtype=torch.int32, device='cuda')
    elif case['call'] in ('lookup', 'scatter'):
        n, v, w = case['tokens'], case['rows'], case['width']
        u = torch.rand(n, device='cuda', dtype=torch.float64, generator=g)
        # uneven frequencies: the density of u^4 on the table; the common tokens lie apart
        at = ((u ** 4 if case['skewed'] else u) * v).long().clamp_(max=v - 1)
        ids = (at * 7919 + seed) % v if math.gcd(7919, v) == 1 else at
        if n > 64:
            ids[::97] = -1  # padding, which has no row
        s['ids'] = ids if case['wide_ids'] else ids.int()
        s['scale'] = math.sqrt(w)
        if case['call'] == 'lookup':
            s['table'] = normal(v, w, scale=0.02)
        else:
            s['dout'] = normal(n, w, scale=0.1)
    else:
        r, w = case['rows'], case['width']
        s['x'], s['residual'], s['dy'] = normal(r, w), normal(r, w), normal(r, w, scale=0.1)
        s['seed'] = 1469598103934665603 + seed  # (more than 32 bits)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    hip, device = _library()
    dtype = {'f32': hip.F32, 'f16': hip.F16, 'bf16': hip.BF16}[case['dtype']]
    s['device'], s['dtype'] = device, dtype
    views = s['views'] = {}
    if case['call'] in ('attend', 'train'):
        b, lq, lk, h, hk, d = (case[k] for k in ('batch', 'queries', 'keys', 'heads', 'kv_heads', 'dim'))
        s['plan'] = hip.Attention(device, dtype, b, lq, lk, h, hk, d, left=case['left'], right=case['right'],
                                  backward=case['call'] == 'train')
        s['out'], s['lse'] = torch.empty_like(s['q']), torch.empty((b, h, lq), device='cuda')
        if case['call'] == 'train':
            s['dq'], s['dk'], s['dv'] = (torch.empty_like(s[k]) for k in 'qkv')
        for k in ('q', 'k', 'v', 'out', 'dout', 'dq', 'dk', 'dv'):
            if k in s:
                views[k] = hip.Heads.of(s[k])
    elif case['call'] in ('lookup', 'scatter'):
        n, v, w = case['tokens'], case['rows'], case['width']
        s['plan'] = hip.Embedding(device, dtype, v, w, n, index_bytes=8 if case['wide_ids'] else 4)
        if case['call'] == 'lookup':
            s['out'] = torch.empty((n, w), device='cuda', dtype=TYPES[case['dtype']])
        else:
            s['dtable'] = torch.empty((v, w), device='cuda')
        for k in ('table', 'out', 'dout', 'dtable'):
            if k in s:
                views[k] = hip.Rows.of(s[k])
    else:
        s['y'], s['dx'] = torch.empty_like(s['x']), torch.empty_like(s['x'])
        for k in ('x', 'residual', 'dy', 'y', 'dx'):
            views[k] = hip.Rows.of(s[k])
    return s


# ----------------------------------------------------------------------------- the plain forms
def _visible(s):
    """[batch, queries, keys]: which keys a query sees."""
    c = s['case']
    i = torch.arange(c['queries'], device='cuda').view(1, -1, 1)
    j = torch.arange(c['keys'], device='cuda').view(1, 1, -1)
    ql = s['ql'].view(-1, 1, 1) if 'ql' in s else torch.full((1, 1, 1), c['queries'], device='cuda')
    kl = s['kl'].view(-1, 1, 1) if 'kl' in s else torch.full((1, 1, 1), c['keys'], device='cuda')
    seen = (i < ql) & (j < kl)
    if c['left'] >= 0:
        seen = seen & (j >= i + kl - ql - c['left'])
    if c['right'] >= 0:
        seen = seen & (j <= i + kl - ql + c['right'])
    return seen


def _plain_attention(s):
    c = s['case']
    b, lq, lk, h, hk, d = (c[k] for k in ('batch', 'queries', 'keys', 'heads', 'kv_heads', 'dim'))
    dtype, scale = s['q'].dtype, 1.0 / math.sqrt(d)

    def rows(x):      # [batch, kv heads, group * queries, dim] in 32 bits
        return x.float().view(b, lq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)

    def unrows(x):
        return x.view(b, hk, h // hk, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, h, d).to(dtype)

    def keys(x):      # [batch, kv heads, keys, dim]
        return x.float().permute(0, 2, 1, 3).contiguous()

    q, k, v = rows(s['q']), keys(s['k']), keys(s['v'])
    score = (q @ k.transpose(-1, -2).contiguous()) * scale
    hidden = ~_visible(s)[:, None, None]
    score = score.view(b, hk, h // hk, lq, lk).masked_fill_(hidden, -math.inf).view(b, hk, -1, lk)
    top = score.amax(-1, keepdim=True)
    score -= torch.where(top == -math.inf, 0.0, top)
    p = score.exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, 1.0, total)
    out = p @ v
    lse = (top + total.log()).view(b, h, lq)
    result = {'out': unrows(out), 'lse': lse}
    if c['call'] == 'train':
        dout = rows(s['dout'])
        result['dv'] = (p.transpose(-1, -2).contiguous() @ dout).permute(0, 2, 1, 3).to(dtype)
        ds = dout @ v.transpose(-1, -2).contiguous()
        ds -= (dout * out).sum(-1, keepdim=True)
        ds *= p
        ds *= scale
        del p, score
        result['dq'] = unrows(ds @ k)
        result['dk'] = (ds.transpose(-1, -2).contiguous() @ q).permute(0, 2, 1, 3).to(dtype)
    return result


def _plain_lookup(s):
    ids = s['ids'].long()
    rows = s['table'][ids.clamp(min=0)].float() * s['scale']
    return {'out': torch.where((ids >= 0)[:, None], rows, 0.0).to(s['table'].dtype)}


def _plain_scatter(s):
    c, ids = s['case'], s['ids'].long()
    dtable = torch.zeros((c['rows'], c['width']), device='cuda')
    rows = torch.where((ids >= 0)[:, None], s['dout'].float() * s['scale'], 0.0)
    return {'dtable': dtable.index_add_(0, ids.clamp(min=0), rows)}


def _product(a, b):
    """High and low 32 bits of the products of a constant and 32-bit words held in 64."""
    low = a * (b & 0xFFFF)
    high = a * (b >> 16) + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _words(count, seed, offset):
    """The generator's words of elements 0..count, in order: four a counter."""
    counter = torch.arange((count + 3) // 4, device='cuda', dtype=torch.int64) + offset
    c0, c1 = counter & 0xFFFFFFFF, counter >> 32
    c2, c3 = torch.zeros_like(counter), torch.zeros_like(counter)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _product(MULTIPLIERS[0], c0)
        h1, l1 = _product(MULTIPLIERS[1], c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + ROUND_KEYS[0]) & 0xFFFFFFFF, (k1 + ROUND_KEYS[1]) & 0xFFFFFFFF
    return torch.stack([c0, c1, c2, c3], -1).view(-1)[:count]


def _plain_dropout(s):
    c = s['case']
    threshold = round(c['probability'] * 2 ** 32)
    keep = (_words(c['rows'] * c['width'], s['seed'], OFFSET) >= threshold).view(c['rows'], c['width'])
    up = 2 ** 32 / (2 ** 32 - threshold)
    dtype = s['x'].dtype
    return {'y': (torch.where(keep, s['x'].float() * up, 0.0) + s['residual'].float()).to(dtype),
            'dx': torch.where(keep, s['dy'].float() * up, 0.0).to(dtype)}


# ----------------------------------------------------------------------------- the calls
def run(s):
    c = s['case']
    if not own:
        return {'attend': _plain_attention, 'train': _plain_attention, 'lookup': _plain_lookup,
                'scatter': _plain_scatter, 'dropout': _plain_dropout}[c['call']](s)
    w = s['views']
    if c['call'] in ('attend', 'train'):
        s['plan'].forward(w['q'], w['k'], w['v'], w['out'], s['lse'], s.get('ql'), s.get('kl'))
        if c['call'] == 'attend':
            return {'out': s['out'], 'lse': s['lse']}
        s['plan'].backward(w['q'], w['k'], w['v'], w['out'], s['lse'], w['dout'], w['dq'], w['dk'], w['dv'],
                           s.get('ql'), s.get('kl'))
        return {'out': s['out'], 'lse': s['lse'], 'dv': s['dv'], 'dq': s['dq'], 'dk': s['dk']}
    if c['call'] == 'lookup':
        s['plan'].forward(s['ids'], c['tokens'], w['table'], w['out'], s['scale'])
        return {'out': s['out']}
    if c['call'] == 'scatter':
        s['plan'].backward(s['ids'], c['tokens'], w['dout'], w['dtable'], s['scale'])
        return {'dtable': s['dtable']}
    s['device'].dropout(s['dtype'], c['rows'], c['width'], w['x'], w['y'], c['probability'], s['seed'], OFFSET,
                        residual=w['residual'])
    s['device'].dropout(s['dtype'], c['rows'], c['width'], w['dy'], w['dx'], c['probability'], s['seed'], OFFSET)
    return {'y': s['y'], 'dx': s['dx']}


# ----------------------------------------------------------------------------- 64 bits
def _exact_attention(s):
    """One head at a time, gradients by automatic differentiation."""
    c = s['case']
    group = c['heads'] // c['kv_heads']
    names = ('q', 'k', 'v')
    grads = {n: torch.zeros(s[n].shape, dtype=torch.float64, device='cuda') for n in names}
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda')
    lse = torch.full((c['batch'], c['heads'], c['queries']), -math.inf, dtype=torch.float64, device='cuda')
    for b, (ql, kl) in enumerate(zip(*_lengths(c))):
        if not ql or not kl:
            continue
        gap = (torch.arange(kl, device='cuda')[None, :] - torch.arange(ql, device='cuda')[:, None]) - (kl - ql)
        hidden = torch.zeros((ql, kl), dtype=torch.bool, device='cuda')
        if c['left'] >= 0:
            hidden |= gap < -c['left']
        if c['right'] >= 0:
            hidden |= gap > c['right']
        empty = hidden.all(1)
        for h in range(c['heads']):
            q, k, v = (s[n][b, :m, h if n == 'q' else h // group].double().requires_grad_(c['call'] == 'train')
                       for n, m in zip(names, (ql, kl, kl)))
            score = torch.matmul(q, k.t()) * c['dim'] ** -0.5
            score = torch.where(hidden, torch.where(empty[:, None], 0.0, -math.inf), score)
            weight = torch.where(empty[:, None], 0.0, torch.softmax(score, 1))
            o = torch.matmul(weight, v)
            out[b, :ql, h] = o.detach()
            lse[b, h, :ql] = torch.where(empty, -math.inf, torch.logsumexp(score.detach(), 1))
            if c['call'] == 'train':
                for n, m, g in zip(names, (ql, kl, kl), torch.autograd.grad(o, (q, k, v), s['dout'][b, :ql, h].double())):
                    grads[n][b, :m, h if n == 'q' else h // group] += g
    if c['call'] == 'attend':
        return {'out': out, 'lse': lse}
    return {'out': out, 'lse': lse, 'dv': grads['v'], 'dq': grads['q'], 'dk': grads['k']}


def _exact_keep(case, seed):
    """The mask from the generator's definition, in numpy on the host."""
    count = case['rows'] * case['width']
    with np.errstate(over='ignore'):
        counter = np.arange(-(-count // 4), dtype=np.uint64) + np.uint64(OFFSET)
        mask, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
        x = [counter & mask, counter >> shift, np.zeros_like(counter), np.zeros_like(counter)]
        key = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            a, b = x[0] * np.uint64(MULTIPLIERS[0]), x[2] * np.uint64(MULTIPLIERS[1])
            x = [(b >> shift) ^ x[1] ^ np.uint64(key[0]), b & mask, (a >> shift) ^ x[3] ^ np.uint64(key[1]), a & mask]
            key = [(k + r) & 0xFFFFFFFF for k, r in zip(key, ROUND_KEYS)]
    keep = np.stack(x, -1).reshape(-1)[:count] >= np.uint64(round(case['probability'] * 2 ** 32))
    return torch.from_numpy(keep.reshape(case['rows'], case['width'])).cuda()


def exact(case, seed):
    s = _inputs(case, seed)
    if case['call'] in ('attend', 'train'):
        return _exact_attention(s)
    if case['call'] == 'lookup':
        padded = torch.cat([s['table'].double() * s['scale'], torch.zeros((1, case['width']), device='cuda')])
        return {'out': padded[torch.where(s['ids'] < 0, case['rows'], s['ids']).long()]}
    if case['call'] == 'scatter':
        padded = torch.zeros((case['rows'] + 1, case['width']), dtype=torch.float64, device='cuda')
        at = torch.where(s['ids'] < 0, case['rows'], s['ids']).long()
        padded.index_put_((at,), s['dout'].double() * s['scale'], accumulate=True)
        return {'dtable': padded[:-1]}
    keep = _exact_keep(case, s['seed']).double()
    up = 1.0 / (1.0 - round(case['probability'] * 2 ** 32) / 2 ** 32)
    return {'y': keep * s['x'].double() * up + s['residual'].double(), 'dx': keep * s['dy'].double() * up}
