"""E2M1 (4-bit) codes of the MX wire format: quantization in one and in both orientations, for any number of rows and for
two formats at once, and the decode, against a plain float64 form; every result is exact."""
import numpy as np
import pytest
import torch

import data_gen
import mx_plain as P

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def tensors():
    rng = np.random.default_rng(7)
    yield "student_t", data_gen.c2_student_t(96, 512, seed=71, as_tensor=True)
    yield "one_row", data_gen.c1_normal(1, 4096, seed=72, as_tensor=True)
    yield "one_block", data_gen.c1_normal(1, 32, seed=73, as_tensor=True)
    yield "ragged_tile", data_gen.c1_normal(160, 224, seed=74, as_tensor=True)
    # every binary exponent, the subnormal and the largest values among them
    wide = (rng.integers(0x0000, 0x7F80, (64, 128)) | (rng.integers(0, 2, (64, 128)) << 15)).astype(np.uint16)
    wide[3] = rng.integers(0x0001, 0x0080, 128)                    # blocks of subnormal values only
    wide[4] = 0x7F7F                                               # the largest value
    wide[5] = 0x8000                                               # negative zeros
    wide[6, :32] = 0
    yield "all_exponents", torch.from_numpy(wide.view(np.int16)).view(torch.bfloat16)
    # every midpoint and every value of the grid, both signs, in blocks of scale 1
    grid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0, 0.5, 1, 1.5, 2, 3, 4, 4.5])
    yield "midpoints", P.bf16(np.tile(np.concatenate([grid, -grid]), (32, 2)))


@pytest.mark.parametrize("case", list(tensors()), ids=lambda c: c[0])
def test_quantize_and_decode(case):
    from mor_amd import wire
    name, x = case
    codes, scales = P.quantize(P.to64(x), P.E2M1)
    p, s = wire.quantize_mx(x.cuda(), wire.E2M1)
    assert np.array_equal(s.cpu().numpy(), scales), name
    assert np.array_equal(p.cpu().numpy(), P.pack(codes, P.E2M1)), name
    got = wire.dequantize_mx(p, s, wire.E2M1)
    want = P.decode(P.pack(codes, P.E2M1), scales, P.E2M1)         # at most two significant bits: exact in bf16 ...
    assert np.array_equal(P.to64(got), P.to64(P.bf16(want))), name  # ... down to its subnormal step


@pytest.mark.parametrize("case", [c for c in tensors() if c[1].shape[0] % 32 == 0], ids=lambda c: c[0])
def test_both_orientations(case):
    from mor_amd import wire
    name, x = case
    rp, rs, cp, cs = wire.quantize_mx_dual(x.cuda(), wire.E2M1)
    for p, s, v in ((rp, rs, x), (cp, cs, x.t())):
        codes, scales = P.quantize(P.to64(v), P.E2M1)
        assert np.array_equal(s.cpu().numpy(), scales), name
        assert np.array_equal(p.cpu().numpy(), P.pack(codes, P.E2M1)), name


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 77, 127, 128, 129, 300])
@pytest.mark.parametrize("fmts", [(P.E4M3, P.E4M3), (P.E5M2, P.E5M2), (P.E2M1, P.E2M1), (P.E2M1, P.E4M3)], ids=str)
def test_both_orientations_of_any_number_of_rows(rows, fmts):
    """The last block of every column is filled up with zeros; nothing is written behind the outputs."""
    from mor_amd import _cabi
    L = _cabi.lib()
    cols = 224
    x = data_gen.c2_student_t(rows, cols, seed=90 + rows, as_tensor=True)
    high = -(-rows // 32) * 32
    want = [P.quantize(P.to64(x), fmts[0]), P.quantize(np.pad(P.to64(x), ((0, high - rows), (0, 0))).T, fmts[1])]
    sizes = [rows * cols * P.BITS[fmts[0]] // 8, rows * cols // 32, cols * high * P.BITS[fmts[1]] // 8, cols * high // 32]
    out = [torch.full((n + 64,), 0xA5, dtype=torch.uint8, device="cuda") for n in sizes]
    xd = x.cuda()
    _cabi.check(L.mor_mx_quantize_dual_ragged(xd.data_ptr(), *[o.data_ptr() for o in out], rows, cols, *fmts, torch.cuda.current_stream().cuda_stream))
    got = [o.cpu().numpy() for o in out]
    for k, (codes, scales) in enumerate(want):
        assert np.array_equal(got[2 * k][: sizes[2 * k]], P.pack(codes, fmts[k]).ravel())
        assert np.array_equal(got[2 * k + 1][: sizes[2 * k + 1]], scales.ravel())
    for g, n in zip(got, sizes):
        assert (g[n:] == 0xA5).all()


def test_blocks_with_infinities_and_nans():
    """E2M1 has no code for them: the block's scale byte is the E8M0 NaN, its codes are 0, it decodes to NaNs; its
    neighbours are not touched."""
    from mor_amd import wire
    x = data_gen.c1_normal(64, 128, seed=75, as_tensor=True)
    for at, v in (((0, 0), float("inf")), ((1, 63), float("-inf")), ((2, 127), float("nan")), ((40, 32), float("nan"))):
        x[at] = v
    p, s = wire.quantize_mx(x.cuda(), wire.E2M1)
    codes, scales = P.quantize(P.to64(x), P.E2M1)
    assert (scales == 255).sum() == 4
    assert np.array_equal(s.cpu().numpy(), scales) and np.array_equal(p.cpu().numpy(), P.pack(codes, P.E2M1))
    got = P.to64(wire.dequantize_mx(p, s, wire.E2M1))
    want = P.decode(P.pack(codes, P.E2M1), scales, P.E2M1)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])
    rp, rs, cp, cs = wire.quantize_mx_dual(x.cuda(), wire.E2M1)
    codes_t, scales_t = P.quantize(P.to64(x.t()), P.E2M1)
    assert torch.equal(rp, p) and torch.equal(rs, s)
    assert np.array_equal(cs.cpu().numpy(), scales_t) and np.array_equal(cp.cpu().numpy(), P.pack(codes_t, P.E2M1))


def test_decode_of_every_code_and_scale():
    from mor_amd import wire
    payload = np.tile((np.arange(16) * 17).astype(np.uint8), (256, 1))       # codes 0 0 1 1 .. 15 15
    scales = np.arange(256, dtype=np.uint8)[:, None]
    got = wire.dequantize_mx(torch.from_numpy(payload).cuda(), torch.from_numpy(scales).cuda(), wire.E2M1)
    want = P.bf16(P.decode(payload, scales, P.E2M1))                          # overflows to infinity at the largest scales
    g, w = P.to64(got), P.to64(want)
    assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(g[~np.isnan(w)], w[~np.isnan(w)])
    assert np.array_equal(np.signbit(g[~np.isnan(w)]), np.signbit(w[~np.isnan(w)]))


def test_hw_converts_selftest():
    """The E2M1 converts against the software codes: 65 280 finite bf16 values x 253 scale exponents, and their inverse."""
    from mor_amd import _cabi
    bad = torch.full((2,), -1, dtype=torch.int64, device="cuda")
    _cabi.check(_cabi.lib().mor_selftest_hw_fp4(bad.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert bad.tolist() == [0, 0]


def test_full_size_properties():
    """8192 x 8192: quantizing the decoded tensor again gives the same values, and the two halves of the dual call equal
    the single call on x and on x transposed."""
    from mor_amd import wire
    x = data_gen.c2_student_t(8192, 8192, seed=1002, as_tensor=True).cuda()
    p, s = wire.quantize_mx(x, wire.E2M1)
    d = wire.dequantize_mx(p, s, wire.E2M1)
    again = wire.dequantize_mx(*wire.quantize_mx(d, wire.E2M1), wire.E2M1)
    assert torch.equal(again.view(torch.int16), d.view(torch.int16))
    rp, rs, cp, cs = wire.quantize_mx_dual(x, wire.E2M1)
    tp, ts = wire.quantize_mx(x.t().contiguous(), wire.E2M1)
    assert torch.equal(rp, p) and torch.equal(rs, s) and torch.equal(cp, tp) and torch.equal(cs, ts)


def test_views_and_streams():
    """A strided view and a tensor that starts at an odd element are copied first; the call runs on the current stream."""
    from mor_amd import wire
    base = data_gen.c1_normal(64, 256, seed=76, as_tensor=True).cuda()
    flat = torch.cat([base.new_zeros(1), base.flatten()])
    shifted = flat[1:].view(64, 256)
    assert shifted.data_ptr() % 16 == 2
    want = wire.quantize_mx(base, wire.E2M1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = wire.quantize_mx(shifted, wire.E2M1)
        half = wire.quantize_mx(base[:, 64:192], wire.E2M1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(half[1], want[1][:, 2:6]) and torch.equal(half[0], want[0][:, 32:96])
