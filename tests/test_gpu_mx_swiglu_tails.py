"""mx.swiglu where exp(-gate) is near the end of fp32: sigmoid(gate) is below the smallest normal fp32 number there, and its
product with up is not, so it has to be kept."""
import numpy as np
import pytest
import torch

import mx_plain as P
import test_gpu_mx_training as base

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def test_gates_from_minus_80_to_the_end_of_exp():
    """fp32's exp(-gate) is finite down to a gate of -88.7.  Relative errors: half a step of bf16 for the one rounding, (|g| + 8)
    2^-22 for the sigmoid in fp32 (see swiglu_forms), and for a subnormal sigmoid half its step of 2^-149."""
    from mor_amd import mx
    gates = np.arange(-88.5, -79.5, 0.5)
    ups = np.array([1.0, -3.0, 1e3, -1e6, 1e20, -2.0 ** 100, 2.0 ** -20])
    g, u = (P.bf16(v) for v in np.meshgrid(gates, ups))
    g64, u64 = P.to64(g), P.to64(u)
    with torch.no_grad():
        h = P.to64(mx.swiglu(g.cuda(), u.cuda()))
    s = 1 / (1 + np.exp(-g64))
    want = g64 * s * u64
    bound = np.abs(want) * (P.BF16_HALF_STEP + (np.abs(g64) + 8) * 2.0 ** -22) + np.abs(g64 * u64) * 2.0 ** -150 + 2.0 ** -133
    assert (np.abs(h - want) <= bound).all()
    assert (h != 0)[np.abs(want) > 2.0 ** -120].all()


def test_gradients_there():
    """-88, -80 and 0.5 are values of E4M3 in one block's scale, so the gradients are those of the formula at the inputs."""
    gates = np.tile([-88.0, -80.0, -88.0, -72.0], 8)[None]
    ups = np.tile([1.0, -2.0, 0.5, 1.5], 8)[None] * 2.0 ** 60
    dh = np.tile([1.0, 4.0, -1.0, 8.0], 8)[None]
    g64, u64, dh64 = gates, ups, dh
    assert np.array_equal(P.quantized_values(g64, P.E4M3), g64) and np.array_equal(P.quantized_values(u64, P.E4M3), u64)
    from mor_amd import mx
    g, u = base.leaf(P.bf16(gates)), base.leaf(P.bf16(ups))
    dg, du = torch.autograd.grad(mx.swiglu(g, u), (g, u), P.bf16(dh).cuda())
    s, rest = 1 / (1 + np.exp(-g64)), 1 / (1 + np.exp(g64))
    want = dh64 * u64 * s * (1 + g64 * rest)
    size = np.abs(dh64 * u64) * (1 + np.abs(g64)) * (s * (1 + np.abs(g64)) * 2.0 ** -20 + 2.0 ** -149)
    assert (np.abs(P.to64(dg) - want) <= P.BF16_HALF_STEP * np.abs(want) + size + 2.0 ** -133).all()
    assert (P.to64(dg) != 0).all()
    want = dh64 * g64 * s
    size = np.abs(dh64 * g64) * (s * (np.abs(g64) + 8) * 2.0 ** -22 + 2.0 ** -149)
    assert (np.abs(P.to64(du) - want) <= P.BF16_HALF_STEP * np.abs(want) + size + 2.0 ** -133).all()
