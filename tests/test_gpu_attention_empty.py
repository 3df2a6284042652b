"""Rows and keys that have no part in a call give zeros whatever stands in the others:
queries past their length or without a key, keys past theirs or without a query, beside
visible keys, values and output gradients that are infinite or NaN."""
import math

import pytest
import torch

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu

SHAPES = [
    (3, 1, 60, 4, 2, 64),        # one and two query rows, short lists and long
    (3, 2, 4000, 4, 4, 32),
    (3, 20, 90, 4, 2, 64),       # one tile of rows
    (3, 24, 3000, 4, 2, 128),    # the same over splits
    (3, 330, 340, 2, 1, 64),     # small sets
    (3, 700, 900, 16, 8, 64),    # many rows and keys
    (3, 100, 8000, 4, 1, 96),
]


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('bad', [math.nan, math.inf])
def test_rows_past_the_lengths(device, dtype, shape, bad):
    """Every entry's first visible key and value are bad, so every row that sees it is; the others are zeros."""
    print(f'[case] past the lengths {dtype} {shape} {bad}', flush=True)
    c = Case(dtype, *shape)
    queries, keys = shape[1:3]
    ql, kl = [queries, queries // 2, queries // 3], [keys, keys - 7, keys // 2]
    c.k[:, 0], c.v[:, 0] = bad, bad
    c.run(device, ql=ql, kl=kl)
    for b in range(3):
        assert (c.out[b, ql[b]:] == 0).all() and (c.lse[b, :, ql[b]:] == -math.inf).all()
        assert (c.dq[b, ql[b]:] == 0).all()
        assert (c.dk[b, kl[b]:] == 0).all() and (c.dv[b, kl[b]:] == 0).all()
        assert not c.out[b, :ql[b]].isfinite().any()


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('queries,keys,heads,kv_heads,dim', [(30, 18, 4, 2, 64), (340, 290, 2, 1, 64), (900, 800, 16, 8, 64),
                                                             (5, 2, 2, 2, 32)])
def test_queries_without_keys(device, dtype, queries, keys, heads, kv_heads, dim):
    """Causal, with more queries than keys: the first queries see none."""
    print(f'[case] no keys {dtype} {queries} x {keys}', flush=True)
    c = Case(dtype, 2, queries, keys, heads, kv_heads, dim)
    c.k[:, 0], c.v[:, 0] = math.nan, math.nan
    c.run(device, right=0)
    none = queries - keys
    assert (c.out[:, :none] == 0).all() and (c.lse[:, :, :none] == -math.inf).all() and (c.dq[:, :none] == 0).all()
    assert c.out[:, none:].isnan().all()


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('queries,keys,heads,kv_heads,dim', [(18, 90, 4, 2, 64), (290, 340, 2, 1, 64), (800, 900, 16, 8, 64),
                                                             (2, 50, 2, 2, 32)])
def test_keys_without_queries(device, dtype, queries, keys, heads, kv_heads, dim):
    """A band that no query's left side reaches past: the first keys are seen by none."""
    print(f'[case] no queries {dtype} {queries} x {keys}', flush=True)
    c = Case(dtype, 2, queries, keys, heads, kv_heads, dim)
    c.dout[:, 0] = math.nan
    c.run(device, left=3, right=0)
    none = keys - queries - 3
    assert (c.dk[:, :none] == 0).all() and (c.dv[:, :none] == 0).all()
    assert c.dv[:, none:keys - queries + 1].isnan().all()
