"""Operands of the MX calls that begin at any byte: copied to an aligned place, as the quantisers copy theirs."""
import numpy as np
import pytest
import torch

import mx_plain as P
import test_gpu_mx_matmul as base

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def shifted(t, by):
    """the same values in a contiguous tensor that begins `by` elements into its memory"""
    return torch.cat([t.new_zeros(by), t.flatten()])[by:].view(t.shape)


@pytest.mark.parametrize("by", [1, 4, 8, 12])
def test_product(by):
    from mor_amd import wire
    rng = np.random.default_rng(by)
    for m, n, k, pair in ((5, 40, 96, (P.E2M1, P.E4M3)), (130, 140, 544, (P.E5M2, P.E2M1))):
        a, b = base.dev(*base.operand(rng, m, k, pair[0], 2)), base.dev(*base.operand(rng, n, k, pair[1], 2))
        want = wire.matmul_mx(*a, *b, *pair)
        assert shifted(a[0], by).data_ptr() % 16 == by
        assert torch.equal(wire.matmul_mx(*[shifted(t, by) for t in a], *b, *pair), want)
        assert torch.equal(wire.matmul_mx(*a, *[shifted(t, by) for t in b], *pair), want)


@pytest.mark.parametrize("fmt", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("by", [1, 4, 8, 12])
def test_decode(fmt, by):
    from mor_amd import wire
    x = torch.randn(7, 96, generator=torch.Generator().manual_seed(by)).to(torch.bfloat16).cuda()
    p, s = wire.quantize_mx(x, fmt)
    assert torch.equal(wire.dequantize_mx(shifted(p, by), shifted(s, by), fmt), wire.dequantize_mx(p, s, fmt))
