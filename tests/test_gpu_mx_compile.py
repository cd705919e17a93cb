"""mx.linear, mx.swiglu and matmul_mx under torch.compile: forward and backward traced, with static and with symbolic sizes,
and run by the kernels themselves (the backends leave the operators as they are)."""
import pytest
import torch

import test_gpu_mx_training as base

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def block(x, gate, up, down):
    from mor_amd import mx, wire
    h = mx.swiglu(mx.linear(x, gate, wire.E2M1), mx.linear(x, up, wire.E2M1, wire.E5M2))
    return mx.linear(h, down)


@pytest.mark.parametrize("dynamic", [False, True])
def test_a_block_forward_and_backward(dynamic):
    weights = [base.leaf(base.randn(i, *s, scale=0.1)) for i, s in enumerate(((96, 64), (96, 64), (64, 96)))]
    torch._dynamo.reset()
    compiled = torch.compile(block, backend="aot_eager", dynamic=dynamic, fullgraph=True)
    for shape in ((45, 64), (70, 64), (2, 19, 64)):
        x, dy = base.leaf(base.randn(9, *shape)), base.randn(10, *shape).cuda()
        want = block(x, *weights)
        got = compiled(x, *weights)
        assert torch.equal(got, want)
        grads = [torch.autograd.grad(y, [x, *weights], dy) for y in (got, want)]
        assert all(torch.equal(a, b) for a, b in zip(*grads))
        with torch.no_grad():
            assert torch.equal(compiled(x, *weights), want)
    torch._dynamo.reset()


@pytest.mark.parametrize("dynamic", [False, True])
def test_products_of_codes(dynamic):
    from mor_amd import wire

    def f(x, w):
        a, sa, _, _ = wire.quantize_mx_dual(x, wire.E2M1)
        b, sb = wire.quantize_mx(w)
        return wire.matmul_mx(a, sa, b, sb, wire.E2M1, wire.E4M3), wire.dequantize_mx(a, sa, wire.E2M1)

    torch._dynamo.reset()
    compiled = torch.compile(f, backend="aot_eager", dynamic=dynamic, fullgraph=True)
    for rows in (32, 64, 160):
        x, w = base.randn(rows, rows, 64).cuda(), base.randn(3, 40, 64).cuda()
        assert all(torch.equal(a, b) for a, b in zip(compiled(x, w), f(x, w)))
    torch._dynamo.reset()
