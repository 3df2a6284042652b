"""Table gradients of sizes whose float64 sums are made on the GPU (torch's, in double)."""
import pytest
import torch

from cpde_amd import hip
from sequences import E, TYPES
from test_gpu_embedding import ids_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype,tokens,rows,width,kind', [
    ('f32', 70001, 63, 512, 'uniform'), ('f32', 70001, 63, 512, 'one'), ('f16', 70001, 1000, 513, 'skewed'),
    ('bf16', 131072, 65536, 512, 'skewed'), ('bf16', 200003, 40, 1024, 'outside')])
def test_gradient(device, dtype, tokens, rows, width, kind):
    print(f'[case] large gradient {dtype} tokens={tokens} rows={rows} width={width} {kind}', flush=True)
    ids = ids_of(kind, tokens, rows)
    dout = torch.empty(tokens, width, device='cuda', dtype=TYPES[dtype][0]).normal_(
        generator=torch.Generator('cuda').manual_seed(2))
    dtable = torch.full((rows, width), float('nan'), device='cuda')
    on = ids.int().cuda()
    plan = hip.Embedding(device, TYPES[dtype][1], rows, width, tokens)
    torch.cuda.synchronize()
    plan.backward(on, tokens, hip.Rows.of(dout), hip.Rows.of(dtable), 1.5)
    device.synchronize()
    plan.destroy()
    at = torch.where((ids >= 0) & (ids < rows), ids, rows).cuda()
    x = dout.double() * 1.5

    def sums(v):
        return torch.zeros(rows + 1, *v.shape[1:], dtype=torch.float64, device='cuda').index_add_(0, at, v)[:rows]

    # a sum's roundings, one an addition, and its product's
    far = (sums(torch.ones(tokens, dtype=torch.float64, device='cuda'))[:, None] + 3) * E * sums(x.abs())
    off = (dtable.double() - sums(x)).abs()
    assert (off <= far).all(), float((off / far.clamp(min=1e-300)).max())
