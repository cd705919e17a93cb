"""What mx.linear and mx.swiglu keep for the backward pass may be packed away by a hook and come back at any address."""
import pytest
import torch

import test_gpu_mx_training as base

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


@pytest.mark.parametrize("by", [0, 1, 8, 12])
def test_kept_codes_moved(by):
    from mor_amd import mx, wire
    x, w, dy = base.leaf(base.randn(1, 45, 64)), base.leaf(base.randn(2, 96, 64)), base.randn(3, 45, 96).cuda()

    def run():
        h = mx.swiglu(*[mx.linear(x, w, wire.E2M1, wire.E5M2)] * 2)
        return h

    def moved(host):
        buffer = torch.empty(host.numel() + by, dtype=torch.uint8, device="cuda")
        buffer[by:] = host
        return buffer[by:]

    want = torch.autograd.grad(run(), (x, w), dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), moved):
        h = run()
    got = torch.autograd.grad(h, (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
