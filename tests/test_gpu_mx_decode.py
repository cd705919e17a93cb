"""The decode of the MX wire format: every code with every scale byte, in every format, against the values themselves."""
import numpy as np
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

E4M3, E5M2, E3M2, E2M3, E2M1 = 0, 1, 2, 3, 4
BITS = {E4M3: 8, E5M2: 8, E3M2: 6, E2M3: 6, E2M1: 4}
SMALL = {E3M2: (3, 2, 3), E2M3: (2, 3, 1), E2M1: (2, 1, 1)}          # exponent bits, mantissa bits, bias


def values(fmt):
    """the float64 value of every code"""
    codes = np.arange(1 << BITS[fmt], dtype=np.uint8)
    if BITS[fmt] == 8:
        return torch.from_numpy(codes).view(torch.float8_e4m3fn if fmt == E4M3 else torch.float8_e5m2).double().numpy()
    e_bits, m_bits, bias = SMALL[fmt]
    e, m = (codes >> m_bits) & ((1 << e_bits) - 1), codes & ((1 << m_bits) - 1)
    v = np.where(e == 0, m * 2.0 ** (1 - bias - m_bits), (1 + m / 2 ** m_bits) * np.exp2(e.astype(float) - bias))
    return np.where(codes >> (BITS[fmt] - 1), -v, v)


def packed(codes, bits):
    """codes [rows, n] -> little-endian bytes [rows, n * bits / 8]"""
    if bits == 8:
        return codes
    if bits == 4:
        return codes[:, 0::2] | (codes[:, 1::2] << 4)
    c = codes.astype(np.uint32).reshape(codes.shape[0], -1, 4)
    w = c[..., 0] | (c[..., 1] << 6) | (c[..., 2] << 12) | (c[..., 3] << 18)
    return np.stack([w & 255, (w >> 8) & 255, w >> 16], -1).astype(np.uint8).reshape(codes.shape[0], -1)


@pytest.mark.parametrize("fmt", sorted(BITS))
def test_every_code_and_scale(fmt):
    """At most four significant bits times a power of two: exact, or one rounding at the ends of bf16's range.  Scale byte
    255 stands for NaN."""
    from mor_amd import wire
    row = np.resize(np.arange(1 << BITS[fmt], dtype=np.uint8), max(1 << BITS[fmt], 32))
    codes = np.tile(row, (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], row.size // 32, 1)
    got = wire.dequantize_mx(torch.from_numpy(packed(codes, BITS[fmt])).cuda(), torch.from_numpy(scales).cuda(), fmt).cpu()
    with np.errstate(over="ignore", invalid="ignore"):
        want = values(fmt)[codes] * np.where(np.arange(256) == 255, np.nan, np.exp2(np.arange(256.0) - 127))[:, None]
    want = torch.from_numpy(want).to(torch.bfloat16)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan) and nan[255].all()
    assert torch.equal(got.view(torch.int16)[~nan], want.view(torch.int16)[~nan])
