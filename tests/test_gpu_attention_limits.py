"""Attention shapes at the limit of what one launch takes (fewer than 2^32 lanes)."""
import pytest
import torch

from cpde_amd import hip

pytestmark = pytest.mark.gpu

LIMIT = 1 << 32


def create(device, batch, queries, keys, heads, kv_heads, dim, backward, dtype=hip.BF16):
    hip.Attention(device, dtype, batch, queries, keys, heads, kv_heads, dim, backward=backward).destroy()


@pytest.mark.parametrize('batch,queries,keys,heads,kv_heads,dim,backward', [
    (LIMIT // 1024, 1, 8, 1, 1, 16, False),    # single tokens, short lists: 1,024 lanes a pair
    (LIMIT // 4096, 1, 8, 8, 4, 16, False),
    (LIMIT // 256, 8, 64, 1, 1, 16, False),    # few rows: at least 128 lanes a pair, in workgroups of 32 rows
    (LIMIT // 256, 128, 128, 1, 1, 16, False),
    (LIMIT // 512, 128, 128, 1, 1, 16, True),  # both gradients' workgroups in one launch
])
def test_refused(device, batch, queries, keys, heads, kv_heads, dim, backward):
    with pytest.raises(hip.CpdeError, match='too many workgroups') as err:
        create(device, batch, queries, keys, heads, kv_heads, dim, backward)
    assert err.value.code == hip.EINVAL


@pytest.mark.parametrize('batch,queries,keys,backward', [
    (LIMIT // 1024 - 1, 1, 8, False), (LIMIT // 512 - 8, 32, 32, False), (LIMIT // 1024, 32, 32, True), (0, 5, 5, True)])
def test_taken(device, batch, queries, keys, backward):
    create(device, batch, queries, keys, 1, 1, 16, backward)


def test_rows_past_the_statistics_lanes(device):
    """2^28 rows, whose statistics take sixteen lanes each: more than one launch has.  With
    one key, out is its value, dq and dk are zeros, and dv is the sum of dout: whole numbers,
    so exact."""
    batch, queries, heads, dim = 4096, 8192, 8, 8
    assert batch * queries * heads * 16 == LIMIT
    g = torch.Generator('cuda').manual_seed(1)
    q = torch.ones(1, 1, 1, dim, device='cuda', dtype=torch.bfloat16).expand(batch, queries, heads, dim)
    k, v, row = (torch.randint(-3, 4, (batch, 1, heads, dim), generator=g, device='cuda').to(torch.bfloat16) for _ in range(3))
    dout = row.expand(batch, queries, heads, dim)
    out, dq = (torch.empty(batch, queries, heads, dim, device='cuda', dtype=torch.bfloat16) for _ in range(2))
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    lse = torch.empty(batch, heads, queries, device='cuda')
    dq.fill_(1)
    plan = hip.Attention(device, hip.BF16, batch, queries, 1, heads, heads, dim)
    torch.cuda.synchronize()
    q_, k_, v_, out_, dout_, dq_, dk_, dv_ = (hip.Heads.of(t) for t in (q, k, v, out, dout, dq, dk, dv))
    plan.forward(q_, k_, v_, out_, lse)
    plan.backward(q_, k_, v_, out_, lse, dout_, dq_, dk_, dv_)
    device.synchronize()
    plan.destroy()
    assert (out == v).all()
    assert (dq == 0).all() and (dk == 0).all()
    # (a probability of 1 within a float's roundings is 1 in 16 bits)
    assert (dv.float() == 8192 * row.float()).all()
