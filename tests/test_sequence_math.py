"""The float64 forms that the operators on sequences are tested against, and the
refusals that need no GPU."""
import ctypes

import numpy as np
import torch

from cpde_amd import hip
import sequences


def test_generator_known_answers():
    """Philox4x32-10's published answer for a counter and key of zeros."""
    words = sequences.philox(np.zeros(1, np.uint64), 0)[0]
    assert [int(w) for w in words] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


def test_kept_share():
    mask = sequences.keep(1000, 1000, 0.1, 42)
    # (five standard deviations of a million draws)
    assert abs(float(mask.double().mean()) - 0.9) < 5 * 3e-4


def test_attention_gradient_by_differentiation():
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(2, n, h, 8, generator=g, dtype=torch.float64, requires_grad=True)
                   for n, h in ((9, 4), (12, 2), (12, 2), (9, 4)))
    ql, kl, left, right = [9, 5], [7, 12], 6, 1
    want = sequences.attention(q, k, v, 0.3, left, right, ql, kl, do)
    total = 0
    for b in range(2):
        seen = sequences.visible(ql[b], kl[b], 9, 12, left, right)
        for h in range(4):
            s = torch.where(seen, 0.3 * q[b, :, h] @ k[b, :, h // 2].T, -1e300)
            p = torch.where(seen, torch.softmax(s, 1), 0.0)
            o = p @ v[b, :, h // 2]
            assert torch.allclose(o, want['out'][0][b, :, h], atol=1e-12)
            total = total + (o * do[b, :, h].detach()).sum()
    for name, grad in zip(('dq', 'dk', 'dv'), torch.autograd.grad(total, (q, k, v))):
        assert torch.allclose(grad, want[name][0], atol=1e-12), name


def test_null_arguments_are_refused_without_a_device():
    lib = hip.load()
    out = ctypes.c_void_p()
    shape = hip.AttentionShape(hip.F32, 1, 1, 1, 1, 1, 32, -1, -1, 0, 0.0)
    assert lib.cpde_attention_create(None, ctypes.byref(shape), ctypes.byref(out)) == hip.EINVAL
    assert lib.cpde_embedding_create(None, hip.F32, 1, 1, 1, 4, ctypes.byref(out)) == hip.EINVAL
    assert lib.cpde_dropout(None, hip.F32, 1, 1, None, None, None, 0.5, 0, 0) == hip.EINVAL
    rows = hip.Rows(None, 0)
    heads = hip.Heads(None, 0, 0, 0)
    assert lib.cpde_attention_forward(None, heads, heads, heads, heads, None, None, None) == hip.EINVAL
    assert lib.cpde_attention_backward(None, heads, heads, heads, heads, None, heads, heads, heads, heads, None,
                                       None) == hip.EINVAL
    assert lib.cpde_embedding_forward(None, None, 0, rows, 1.0, rows) == hip.EINVAL
    assert lib.cpde_embedding_backward(None, None, 0, rows, 1.0, rows, 0) == hip.EINVAL
    assert lib.cpde_attention_destroy(None) == hip.OK
    assert lib.cpde_embedding_destroy(None) == hip.OK
