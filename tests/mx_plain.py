"""Plain float64 forms of the MX wire format and of the operators on it, for the tests of the kernels.

Codes come from a table of the format's values: the nearest one, the even code on a midpoint."""
import numpy as np
import torch

E4M3, E5M2, E2M1 = 0, 1, 4
MANT_BITS = {E4M3: 3, E5M2: 2, E2M1: 1}
EMIN = {E4M3: -6, E5M2: -14, E2M1: 0}
FMAX = {E4M3: 448.0, E5M2: 57344.0, E2M1: 6.0}
BITS = {E4M3: 8, E5M2: 8, E2M1: 4}
BF16_HALF_STEP = 2.0 ** -8          # torch.finfo(torch.bfloat16).eps / 2


def table(fmt):
    """the values of the non-negative codes 0, 1, ... up to the largest"""
    m, e = MANT_BITS[fmt], EMIN[fmt]
    v = [k * 2.0 ** (e - m) for k in range(1 << m)]
    while v[-1] < FMAX[fmt]:
        v += [2.0 ** e * (1 + k / (1 << m)) for k in range(1 << m)]
        e += 1
    return np.array([x for x in v if x <= FMAX[fmt]])


def quantize(x, fmt):
    """float64 [rows, cols] (bf16 values) -> (codes uint8 [rows, cols], scales uint8 [rows, cols / 32])"""
    t = table(fmt)
    b = x.reshape(x.shape[0], -1, 32)
    amax = np.abs(b).max(-1)
    with np.errstate(all="ignore"):
        ratio = (np.float32(FMAX[fmt]) / amax.astype(np.float32)).astype(np.float32)
    e8 = ((ratio.view(np.uint32) >> 23) & 0xFF).astype(np.int64) - 127
    e8 = np.where(amax > 0, np.clip(e8, -127, 127), 0)
    finite = np.isfinite(amax)
    y = np.where(finite[..., None], np.ldexp(np.abs(np.where(finite[..., None], b, 0.0)), e8[..., None]), 0.0)
    mid = (t[1:] + t[:-1]) / 2
    code = np.searchsorted(mid, y, side="left")               # a midpoint goes to the lower neighbour ...
    tie = (code < len(mid)) & (y == mid[np.minimum(code, len(mid) - 1)]) & (code % 2 == 1)
    code = code + tie                                         # ... unless that one is odd
    code = code | np.where(np.signbit(b) & finite[..., None], 1 << (BITS[fmt] - 1), 0)
    scale = np.where(finite, 127 - e8, 255)
    return code.astype(np.uint8).reshape(x.shape), scale.astype(np.uint8)


def pack(codes, fmt):
    return codes if BITS[fmt] == 8 else codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(payload, fmt):
    if BITS[fmt] == 8:
        return payload
    return np.stack([payload & 15, payload >> 4], -1).reshape(payload.shape[0], -1)


def decode(payload, scales, fmt):
    """payload and scale bytes -> float64 values (NaN codes and scale byte 255 give NaN)"""
    c = unpack(payload, fmt).astype(np.int64)
    top = 1 << (BITS[fmt] - 1)
    t, mag = table(fmt), c & (top - 1)
    v = np.where(mag < len(t), t[np.minimum(mag, len(t) - 1)], np.nan) * np.where(c & top, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(*scales.shape, 32) * s[..., None]).reshape(c.shape)


def quantized_values(x, fmt):
    """float64 [rows, any] -> the values of its blocks along rows, the last block filled up with zeros"""
    pad = -x.shape[1] % 32
    full = np.pad(x, ((0, 0), (0, pad)))
    codes, scales = quantize(full, fmt)
    return decode(pack(codes, fmt), scales, fmt)[:, : x.shape[1]]


def to64(t):
    return t.detach().cpu().double().numpy()


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16)


def product_bound(a, b, exact_products=False):
    """(exact product, largest allowed difference) of bf16 results of a b^T for float64 operands (values of codes).

    One rounding to bf16, and the sum in fp32.  Of 8-bit codes the matrix instruction adds eight neighbouring products at
    a time, each cut (toward zero) to multiples of 2^-14 of the largest one's power of two: with 448 * 6 and -448 * 6 among
    the eight, the other six of 0.15625 count 0.125 each and those below 0.125 nothing.  The largest, of at most 8
    significant bits, loses nothing and the seven others less than 7 * 2^-14 of it together, so less than 4.3e-4 of the
    eight's sum of magnitudes.  Products of two 4-bit codes are multiples of 1/4 up to 36: 2^-14 * 32 is below their unit,
    they lose nothing.  The additions of the instructions' sums round by at most (k / 64 + 2) 2^-23 of the sum of magnitudes."""
    want, mags = a @ b.T, np.abs(a) @ np.abs(b).T
    k = a.shape[1]
    summed = (k / 64 + 2) * 2.0 ** -23 + (0.0 if exact_products else 7 * 2.0 ** -14)
    return want, BF16_HALF_STEP * np.abs(want) + (1 + BF16_HALF_STEP) * summed * mags + 2.0 ** -133
