"""Every kernel of the products, in each order of operands and each type, on shapes that reach
it by the plan's own account of its launches, against double on the GPU."""
import math
import re

import pytest
import torch

from cpde_amd import hip
from layers import linear, linear_gradient
from sequences import check
from test_gpu_linear import forward, matrix, operands, plan_of, refused, rows_of

pytestmark = pytest.mark.gpu

# rows, inputs, outputs, whether matrices start at whole 16 bytes: ends inside tiles everywhere
SHAPES = [(4090, 4088, 4080, True), (4091, 4093, 4095, True),      # the largest tiles, straight and from copies
          (2050, 2056, 2064, True), (2051, 2047, 2049, True),      # the next, split in floats
          (2599, 2559, 2601, True), (3300, 3304, 3312, True),      # and not
          (8200, 1032, 1040, True), (1032, 8200, 1040, True), (1032, 1032, 4104, True),  # split in 16 bits: dW, forward, dx
          (1030, 1032, 1040, True), (1032, 4104, 520, True), (520, 1032, 4104, True),    # 64 x 64
          (20000, 72, 136, True), (20000, 71, 137, True),          # its longest inner axes
          (1030, 1032, 1040, False), (2050, 2056, 2064, False),    # through registers for their addresses
          (1032, 8200, 1040, False), (1040, 1032, 8200, False), (700, 12001, 700, True),
          (999, 1203, 1301, True), (300, 4100, 1100, False), (300, 1100, 4100, False),   # and widths
          (70, 200, 136, True), (70, 203, 141, True)]              # few tiles


def ran(plan, rows, aligned):
    """{product: (kernel, side, whether split, how operands come)}"""
    text = plan.info(rows, aligned)
    found = {}
    for part in text.split(', '):
        m = re.fullmatch(r'(\w+) (\w+) (\d+) splits (\d+)( through registers| copied)?', part)
        found[m[1]] = (m[2], int(m[3]), int(m[4]) > 1, (m[5] or '').strip())
    return found, text


def test_shapes_reach_every_kernel(device):
    want = {('product_run_k', 32, False, ''), ('product_run_k', 32, False, 'through registers'),
            ('product_k', 64, False, ''), ('product_k', 64, True, ''), ('product_k', 64, False, 'through registers'),
            ('product_k', 64, True, 'through registers'), ('product_k', 128, False, ''), ('product_k', 128, True, ''),
            ('product_k', 128, False, 'copied'), ('product_large_k', 256, False, ''), ('product_large_k', 256, False, 'copied')}
    for dtype in ('f32', 'f16', 'bf16'):
        seen = {'forward': set(), 'dx': set(), 'dweight': set()}
        for rows, inputs, outputs, aligned in SHAPES:
            plan = plan_of(device, dtype, rows, inputs, outputs, 'none')
            found, text = ran(plan, rows, aligned)
            print(f'[case] {dtype} {rows}x{inputs}x{outputs} {aligned}: {text}', flush=True)
            plan.destroy()
            for product, kernel in found.items():
                seen[product].add(kernel)
        for product, kernels in seen.items():
            assert want <= kernels, (dtype, product, want - kernels)


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('kind', ['none', 'gelu'])
@pytest.mark.parametrize('rows,inputs,outputs,aligned', SHAPES)
def test_values_and_gradients(device, dtype, kind, rows, inputs, outputs, aligned):
    """Within the worst case of each element, and on the whole as near as the type: floats as float
    sums of floats (2e-6 of the norm; sums of up to 20,000 terms round to 2^-24 sqrt(20,000) / 2 =
    4e-6 at most where they are one chain: 32 splits, or 256 rows' strips, cut it under a tenth),
    16-bit results whose operands are not rounded as their exact values rounded once."""
    print(f'[case] linear {dtype} {rows}x{inputs}x{outputs} {kind} aligned={aligned}', flush=True)
    offset = 0 if aligned else 1
    x, w, b, r = operands(dtype, rows, inputs, outputs, True, True, 0, offset)
    plan = plan_of(device, dtype, rows, inputs, outputs, kind)
    dy = matrix(rows, outputs, dtype, 0, offset, 5, 0.1)
    y, z = forward(device, plan, x, w, b, r)
    dx, dw, db = (torch.full(t.shape, math.nan, device='cuda', dtype=t.dtype) for t in (x, w, b))
    torch.cuda.synchronize()
    plan.backward(rows, rows_of(x), rows_of(w), rows_of(dy), pre=rows_of(z) if kind != 'none' else None, dx=rows_of(dx),
                  dweight=rows_of(dw), dbias=db.data_ptr())
    device.synchronize()
    plan.destroy()

    def held(got, values, bounds, name, once):
        check(got, values.cpu(), bounds.cpu(), name)
        least = float((values.to(got.dtype).double() - values).norm() / values.norm())
        far = float((got.double() - values).norm() / values.norm())
        if dtype == 'f32':
            assert far < 2e-6, (name, far)
        elif once:
            assert far < 1.01 * least + 1e-5, (name, far, least)

    want = linear(x, w, b, r, kind, dtype)
    held(y, *want['y'], 'y', True)
    held(z, *want['pre'], 'pre', True)
    want = linear_gradient(x, w, z, dy, kind, dtype)
    held(dx, *want['dx'], 'dx', kind == 'none')
    held(dw, *want['dweight'], 'dweight', kind == 'none')
    check(db, *(t.cpu() for t in want['dbias']), 'dbias')


def test_info_refusals(device):
    plan = hip.Linear(device, hip.F32, 8, 8, 8)
    refused('more rows', lambda: plan.info(9))
    refused('more rows', lambda: plan.info(-1))
    refused('null argument', lambda: hip.check(hip.load().cpde_linear_info(None, 1, 1, None, 0)))
    assert plan.info(0) == 'forward nothing, dx nothing, dweight product_run_k 32 splits 1'
    text = hip.ctypes.create_string_buffer(8)
    hip.check(hip.load().cpde_linear_info(plan.handle, 8, 1, text, 8))
    assert text.value == b'forward'
    plan.destroy()
