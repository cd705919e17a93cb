"""The MX calls say what they refuse when a tensor is in host memory."""
import pytest
import torch

from mor_amd import mx, wire


def test_messages():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16, requires_grad=True)
    p, s = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for call in (lambda: wire.quantize_mx(x), lambda: wire.quantize_mx(x, wire.E2M1), lambda: wire.quantize_mx_dual(x),
                 lambda: wire.dequantize_mx(p, s), lambda: wire.matmul_mx(p, s, p, s), lambda: mx.linear(x, w),
                 lambda: mx.linear(x, w.detach()), lambda: mx.swiglu(x, x), lambda: mx.swiglu(x, w[:4]),
                 lambda: torch.ops.mor.mx_linear_forward(x, w, 0, True, True), lambda: torch.ops.mor.swiglu_mx_backward(x, p)):
        with pytest.raises(RuntimeError, match="mor: .*GPU"):
            call()
