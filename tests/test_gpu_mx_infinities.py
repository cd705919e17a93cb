"""What infinities and NaNs become in the 8-bit formats of the MX wire, and in a product of them."""
import numpy as np
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

E4M3, E5M2 = 0, 1
INF, NAN = float("inf"), float("nan")


def bits(t):
    return t.cpu().view(torch.int16)


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_codes_and_decode(fmt):
    """An infinity takes its block's other values to zero (the scale is the largest); a NaN does not touch them."""
    from mor_amd import wire
    x = torch.randn(64, 96, generator=torch.Generator().manual_seed(fmt)).to(torch.bfloat16)
    clean = wire.dequantize_mx(*wire.quantize_mx(x.cuda(), fmt), fmt).cpu()
    x[3, 5], x[3, 40], x[7, 70], x[40, 33] = INF, -INF, NAN, INF
    calls = [(wire.quantize_mx(x.cuda(), fmt), x, clean)]
    both = wire.quantize_mx_dual(x.cuda(), fmt)
    calls.append((both[:2], x, clean))
    for (p, s), v, plain in calls:
        got = wire.dequantize_mx(p, s, fmt).cpu()
        if fmt == E5M2:
            assert got[3, 5] == INF and got[3, 40] == -INF and got[40, 33] == INF
        else:
            assert torch.isnan(got[[3, 3, 40], [5, 40, 33]]).all()
        assert torch.isnan(got[7, 70])
        special = ~torch.isfinite(v)
        block = special.view(64, 3, 32).any(-1, keepdim=True).expand(64, 3, 32).reshape(64, 96)
        infinite = torch.isinf(v).view(64, 3, 32).any(-1, keepdim=True).expand(64, 3, 32).reshape(64, 96)
        assert (got[infinite & ~special] == 0).all()
        assert torch.equal(bits(got[~block]), bits(plain[~block]))
        assert torch.isfinite(got[block & ~infinite & ~special]).all()
    tp, ts = wire.quantize_mx(x.t().contiguous()[:, :64].contiguous().cuda(), fmt)
    assert torch.equal(both[2], tp) and torch.equal(both[3], ts)


@pytest.mark.parametrize("shape", [(2, 40, 64), (70, 90, 96), (300, 200, 1056)], ids=str)
def test_infinities_of_e5m2_in_a_product(shape):
    """One infinity in a row of a: the row is infinite where b's value is not zero, NaN where it is, and NaN beside one of
    the other sign.  The codes of b are 1, -1 and 0, so every other sum is exact."""
    from mor_amd import wire
    m, n, k = shape
    rng = np.random.default_rng(k)
    a, b = (rng.integers(0, 3, (r, k)) - 1.0 for r in (m, n))
    a[0, 7], a[m - 1, k - 1], a[m // 2, 3] = INF, -INF, INF
    if m > 2:
        a[m // 2, 9] = INF
    enc = lambda v: torch.from_numpy(v).to(torch.float8_e5m2).view(torch.uint8).cuda()  # noqa: E731
    ones = lambda r: torch.full((r, k // 32), 127, dtype=torch.uint8, device="cuda")  # noqa: E731
    got = wire.matmul_mx(enc(a), ones(m), enc(b), ones(n), E5M2).double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = np.stack([(row * b).sum(1) for row in a])
    want = torch.from_numpy(want).to(torch.bfloat16).double().numpy()
    assert np.array_equal(got, want, equal_nan=True)
