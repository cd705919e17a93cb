"""mx.swiglu on tensors past the sizes at which it goes past the caches (2^25, 2^26 and 2^27 elements), and past 2^31."""
import numpy as np
import pytest
import torch

import mx_plain as P
import test_gpu_mx_training as base

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def halves(rows, cols, seed, pad=0):
    """gate and up as the halves of one projection (`pad` elements between them), and a gradient"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    both = torch.empty(rows, 2 * cols + pad, dtype=torch.bfloat16, device="cuda").normal_(0, 3, generator=g)
    dh = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(0, 0.01, generator=g)
    return both[:, :cols], both[:, cols + pad:], dh


def kept_parts(kept, rows, cols):
    """codes and scale bytes of gate and of up, as rows"""
    n, blocks = rows * cols, rows * cols // 32
    up = -(-n // 256) * 256
    at = (0, up, 2 * up, 2 * up + blocks)
    return [kept[a:a + c].view(rows, -1) for a, c in zip(at, (n, n, blocks, blocks))]


@pytest.mark.parametrize("rows", [2050, 4100, 8200])
def test_every_size_class_gives_the_bits_of_small_tensors(rows):
    """Row slices below 2^25 elements, whose loads and stores are plain, against the whole: result, gradients, codes and
    scale bytes."""
    op = torch.ops.mor
    cols = 16384
    gate, up, dh = halves(rows, cols, rows)
    assert gate.stride(0) == 2 * cols and rows * cols > {2050: 1 << 25, 4100: 1 << 26, 8200: 1 << 27}[rows]
    h, kept = op.swiglu_mx_forward(gate, up, True)
    dg, du = op.swiglu_mx_backward(dh, kept)
    parts = kept_parts(kept, rows, cols)
    for r in range(0, rows, 2000):
        cut = slice(r, min(r + 2000, rows))
        hs, ks = op.swiglu_mx_forward(gate[cut], up[cut], True)
        dgs, dus = op.swiglu_mx_backward(dh[cut], ks)
        assert torch.equal(hs, h[cut]) and torch.equal(dgs, dg[cut]) and torch.equal(dus, du[cut]), r
        assert all(torch.equal(a, b[cut]) for a, b in zip(kept_parts(ks, cut.stop - r, cols), parts)), r
    assert torch.equal(op.swiglu_mx_forward(gate, up, False)[0], h)


@pytest.mark.parametrize("cols, pad", [(32800, 0), (32801, 3)], ids=str)
def test_past_2_to_the_31_elements(cols, pad):
    """Rows at the ends and on both sides of elements 2^31 and 2^32 (of the projection) against float64."""
    from mor_amd import mx
    rows = 65600
    assert rows * cols > 1 << 31
    gate, up, dh = halves(rows, cols, 5, pad)
    gate, up = gate.detach().requires_grad_(), up.detach().requires_grad_()
    h = mx.swiglu(gate, up)
    dg, du = torch.autograd.grad(h, (gate, up), dh)
    near = [(1 << 31) // cols, (1 << 32) // (2 * cols + pad), (1 << 31) // (2 * cols + pad)]
    at = torch.tensor(sorted({0, 1, rows - 2, rows - 1} | {r + d for r in near for d in (-1, 0, 1)}), device="cuda")
    at = at[at < rows]
    forms = base.swiglu_forms(*[P.to64(t[at]) for t in (gate, up, dh)])
    for got, (want, bound) in zip((h, dg, du), forms):
        assert (np.abs(P.to64(got[at]) - want) <= bound).all()
