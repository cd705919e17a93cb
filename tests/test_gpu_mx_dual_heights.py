"""wire.quantize_mx_dual for heights that are no multiple of a block and for two formats at once."""
import numpy as np
import pytest
import torch

import data_gen
import mx_plain as P

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


@pytest.mark.parametrize("rows", [0, 1, 31, 32, 33, 129])
@pytest.mark.parametrize("fmts", [(P.E4M3, None), (P.E5M2, P.E5M2), (P.E2M1, None), (P.E2M1, P.E4M3)], ids=str)
def test_codes(rows, fmts):
    from mor_amd import wire
    cols = 96
    x = data_gen.c2_student_t(max(rows, 1), cols, seed=rows, as_tensor=True)[:rows]
    out = wire.quantize_mx_dual(x.cuda(), *fmts)
    high, row_fmt = -(-rows // 32) * 32, fmts[0]
    col_fmt = row_fmt if fmts[1] is None else fmts[1]
    assert [tuple(t.shape) for t in out] == [(rows, cols * P.BITS[row_fmt] // 8), (rows, 3), (cols, high * P.BITS[col_fmt] // 8), (cols, high // 32)]
    if rows:
        columns = np.pad(P.to64(x), ((0, high - rows), (0, 0))).T
        for (p, s), v, fmt in ((out[:2], P.to64(x), row_fmt), (out[2:], columns, col_fmt)):
            codes, scales = P.quantize(v, fmt)
            assert np.array_equal(s.cpu().numpy(), scales) and np.array_equal(p.cpu().numpy(), P.pack(codes, fmt))


def test_weight_gradient_of_a_ragged_batch():
    """The product that they are for: dy^T x over 45 tokens, the zeros adding nothing."""
    from mor_amd import wire
    x, dy = data_gen.c1_normal(45, 64, seed=1, as_tensor=True), data_gen.c1_normal(45, 96, seed=2, as_tensor=True)
    _, _, a, sa = wire.quantize_mx_dual(dy.cuda())
    _, _, b, sb = wire.quantize_mx_dual(x.cuda(), wire.E2M1, wire.E4M3)
    want, bound = P.product_bound(P.quantized_values(P.to64(dy).T, P.E4M3), P.quantized_values(P.to64(x).T, P.E4M3))
    assert (np.abs(P.to64(wire.matmul_mx(a, sa, b, sb)) - want) <= bound).all()


def test_refusals():
    from mor_amd import wire
    x = torch.zeros(33, 64, dtype=torch.bfloat16, device="cuda")
    for fmts in ((wire.E2M3,), (wire.E3M2,), (wire.E4M3, wire.E2M1), (wire.E4M3, wire.E5M2), (7,)):
        with pytest.raises(RuntimeError, match="format"):
            wire.quantize_mx_dual(x, *fmts)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        wire.quantize_mx_dual(x[:, :48])
    with pytest.raises(RuntimeError, match="bfloat16"):
        wire.quantize_mx_dual(x.float())


@pytest.mark.parametrize("shape", [(8192, 8192), (12301, 8192), (16384, 8192), (16416, 8192)], ids=str)
@pytest.mark.parametrize("fmts", [(P.E4M3, None), (P.E2M1, P.E4M3)], ids=str)
def test_every_size_class_gives_the_bits_of_the_single_calls(shape, fmts):
    """Inputs below 192 MiB, of 192 to 256 MiB (read past the caches) and beyond: the halves of the call against
    quantize_mx on x and on x transposed, its rows filled up with zeros."""
    from mor_amd import wire
    rows, cols = shape
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    got = wire.quantize_mx_dual(x, *fmts)
    want = wire.quantize_mx(x, fmts[0])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    high = -(-rows // 32) * 32
    want = wire.quantize_mx(torch.nn.functional.pad(x.t(), (0, high - rows)).contiguous(), fmts[0] if fmts[1] is None else fmts[1])
    assert torch.equal(got[2], want[0]) and torch.equal(got[3], want[1])
