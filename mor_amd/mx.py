"""Training on the MX wire format: a linear layer whose three products are taken in 8 or 4 bits and whose activation is
kept in 8, and a gated activation that keeps its inputs in 8 bits.

The reference simulates this with its callers' torch products on dequantized tensors (mor/ops.py); here the products read
the codes (wire.matmul_mx).  A block is 32 consecutive elements along the axis a product sums over, with the power-of-two
scale of wire.quantize_mx.  Gradients pass straight through the quantisers, as in mor.ops.
"""
import torch
from torch import Tensor

from . import wire

_op = torch.ops.mor


def linear(x: Tensor, weight: Tensor, fmt: int = wire.E4M3, grad_fmt: int = wire.E4M3) -> Tensor:
    """y = Q(x) Q(weight)^T for bfloat16 x [..., inputs] and weight [outputs, inputs] -> bfloat16 [..., outputs].

    Q quantises to blocks along the summed axis: x and weight to `fmt` (E4M3 or E2M1) in the forward product, the
    gradient dy to `grad_fmt` (E4M3 or E5M2) in both backward products:
        dx = Q(dy) Q(weight^T)^T,  weight^T in fmt, blocks along the outputs
        dw = Q(dy^T) Q(x^T)^T,     x^T in E4M3 whatever fmt is, blocks along the tokens (the last one filled up with zeros)
    x^T and weight^T are quantised in the forward pass, from the same read as their other orientation, and are all that
    is kept of x and weight: 1.03 bytes per element of x.  inputs and outputs are multiples of 32, the number of tokens
    is any up to 2^23 - 32, zero included.  There is no second derivative and no forward-mode one: a call with a tangent is refused."""
    if x.dim() == 2:
        return _op.mx_linear(x, weight, fmt, grad_fmt)
    if x.dim() < 2:
        raise RuntimeError(f"mor: x must have at least two dimensions, got {tuple(x.shape)}")
    return _op.mx_linear(x.reshape(-1, x.shape[-1]), weight, fmt, grad_fmt).view(*x.shape[:-1], weight.shape[0])


def swiglu(gate: Tensor, up: Tensor) -> Tensor:
    """gate * sigmoid(gate) * up of two bfloat16 tensors of one shape [..., n] (any n), computed in fp32.

    For the backward pass gate and up are kept as E4M3 codes with a scale byte per 32 elements of a row, written by the
    forward kernel: 2.0625 bytes per pair of elements instead of 4 in bf16.  The gradients are
    those of the formula at the decoded values.  A block that holds an infinity or a NaN comes back as NaNs.  Rows may
    lie at any stride (the halves of one projection are read in place).  There is no second derivative and no
    forward-mode one: a call with a tangent is refused."""
    if gate.shape != up.shape:
        raise RuntimeError(f"mor: gate and up must have one shape, got {tuple(gate.shape)} and {tuple(up.shape)}")
    if gate.dim() == 2:
        return _op.swiglu_mx(gate, up)
    if gate.dim() < 1:
        raise RuntimeError("mor: gate and up must have at least one dimension")
    n = gate.shape[-1]
    rows = gate.numel() // n if n else 0
    return _op.swiglu_mx(gate.reshape(rows, n), up.reshape(rows, n)).view(gate.shape)
