"""Products of MX tensors at the ends of the scales: sums in fp32's subnormal range, below it and past its largest value."""
import pytest
import torch

import mx_plain as P

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

ONE = {P.E4M3: 0x38, P.E5M2: 0x3C, P.E2M1: 0x22}                 # the code of 1 (E2M1: two of them)


@pytest.mark.parametrize("pair", [(P.E4M3, P.E4M3), (P.E2M1, P.E2M1), (P.E4M3, P.E2M1), (P.E5M2, P.E4M3)], ids=str)
@pytest.mark.parametrize("shape", [(16, 16, 32), (64, 64, 64), (300, 300, 1024), (1000, 4001, 1056), (4100, 4601, 96), (100, 64, 14336)], ids=str)
def test_sums_of_equal_powers_of_two(shape, pair):
    """k products of 2^(a + b - 254): exact in fp32 wherever one product is at least 2^-149, so the result is their sum
    rounded once to bf16, down to its subnormal step of 2^-133; zero where all k are below 2^-150 / k; infinite past fp32."""
    from mor_amd import wire
    m, n, k = shape
    codes = lambda rows, fmt: torch.full((rows, k * P.BITS[fmt] // 8), ONE[fmt], dtype=torch.uint8, device="cuda")  # noqa: E731
    scales = lambda rows, byte: torch.full((rows, k // 32), byte, dtype=torch.uint8, device="cuda")  # noqa: E731
    pa, pb = codes(m, pair[0]), codes(n, pair[1])
    for a, b in ((127, 0), (0, 127), (64, 64), (64, 63), (60, 60), (64, 56), (60, 57), (58, 57), (0, 105), (0, 0), (1, 64), (254, 100), (254, 0), (200, 180), (254, 254)):
        want = torch.tensor(k * 2.0 ** (a + b - 254), dtype=torch.float64).to(torch.bfloat16).cuda()
        got = wire.matmul_mx(pa, scales(m, a), pb, scales(n, b), *pair)
        assert (got == want).all(), (a, b, float(want), float(got[0, 0]))
