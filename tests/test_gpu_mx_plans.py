"""Products of MX tensors at the sizes that take the remaining kernels and launches: a last round of large tiles cut off
into small ones along either side, tiles of 128 in eight waves, few rows with k shared by any number of waves.
test_mx_plans.py checks, without a GPU, that with these every kind of plan is among the tested sizes."""
import numpy as np
import pytest
import torch

import mx_plain as P
import test_gpu_mx_matmul as base

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

A8, B8, C4 = P.E4M3, P.E5M2, P.E2M1
EACH = [(A8, A8), (C4, C4), (A8, C4)]
CASES = [(s, p) for s in (
    # columns cut (odd rows of the output, and rows of 16-byte pieces), rows cut
    (4100, 4601, 96), (4100, 4600, 96), (66000, 200, 96),
    # few rows, k in 3, 4 and 8 parts of one or two groups; 512 workgroups and more
    (3, 50, 1344), (5, 9001, 2080), (16, 33, 5152)) for p in EACH] + [
    # the same with the rest in tiles of 64, of 128 in four and in eight waves, which differ with the formats
    ((1281, 11206, 32), (A8, A8)), ((308, 35560, 32), (C4, B8)), ((291, 37118, 32), (C4, C4)),
    ((838, 19949, 160), (B8, A8)), ((277, 42762, 192), (A8, C4)),
    ((41378, 284, 32), (A8, A8)), ((41221, 310, 32), (A8, C4)), ((46854, 303, 32), (C4, C4)),
    ((33038, 289, 96), (A8, C4)), ((38389, 378, 256), (A8, B8)), ((38233, 447, 192), (C4, A8)),
    # tiles of 128 in eight waves, k whole and split
    ((1000, 4001, 1056), (A8, A8)), ((1000, 4001, 1056), (B8, C4)), ((1024, 4096, 4096), (A8, A8)), ((1024, 4096, 4096), (C4, A8)),
    ((88, 3795, 15008), (A8, C4)), ((2308, 205, 15040), (A8, A8)),
    # the rest of the shares of k
    ((2, 70, 2528), (A8, A8)), ((2, 70, 3040), (A8, C4)), ((2, 70, 3552), (C4, C4)),
    ((2, 70, 2528), (C4, C4)), ((2, 70, 3040), (C4, C4)), ((2, 70, 2528), (A8, C4)), ((2, 70, 3040), (A8, A8)), ((2, 70, 3552), (A8, A8)),
    ((2, 70, 3552), (A8, C4)), ((7, 40, 832), (C4, C4)), ((7, 40, 832), (A8, A8)), ((7, 40, 832), (A8, C4))]


def ids(v):
    return base.ids(v)


@pytest.mark.parametrize("shape, pair", CASES, ids=ids)
def test_one_code_per_row_gives_exact_products(shape, pair):
    """Each row of a has one non-zero code: a result is one product of two codes and two scales, exact in bf16."""
    m, n, k = shape
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    (pa, sa), (pb, sb) = base.operand(rng, m, k, pair[0], 20), base.operand(rng, n, k, pair[1], 20)
    at = (np.arange(m) * 37 + rng.integers(0, 5)) % k
    ca = P.unpack(pa, pair[0])
    keep = np.zeros_like(ca)
    keep[np.arange(m), at] = ca[np.arange(m), at]
    pa = P.pack(keep, pair[0])
    va, vb = P.decode(pa, sa, pair[0]), P.decode(pb, sb, pair[1])
    got = base.run((pa, sa), (pb, sb), pair)
    rows = max(1, (1 << 23) // n)
    for r in range(0, m, rows):                                # a few rows at a time: float64 of all of them is large
        i = np.arange(r, min(r + rows, m))
        want = va[i, at[i]][:, None] * vb[:, at[i]].T
        assert np.array_equal(P.to64(got[r:r + rows]), want), r


@pytest.mark.parametrize("shape, pair", CASES, ids=ids)
def test_full_rows(shape, pair):
    m, n, k = shape
    rng = np.random.default_rng(m + n + k)
    a, b = base.operand(rng, m, k, pair[0], 3), base.operand(rng, n, k, pair[1], 3)
    got = base.run(a, b, pair)
    va, vb = P.decode(*a, pair[0]), P.decode(*b, pair[1])
    rows = max(1, (1 << 23) // n)
    for r in range(0, m, rows):
        want, bound = P.product_bound(va[r:r + rows], vb, exact_products=pair == (C4, C4))
        assert (np.abs(P.to64(got[r:r + rows]) - want) <= bound).all(), r


@pytest.mark.parametrize("shape, pair", [((4100, 4601, 96), (A8, A8)), ((4100, 4600, 96), (C4, C4)), ((66000, 200, 96), (A8, C4)),
                                         ((838, 19949, 160), (A8, A8)), ((2308, 205, 15040), (A8, A8))], ids=ids)
def test_nothing_behind_the_output_or_the_workspace_is_written(shape, pair):
    from mor_amd import _cabi
    L = _cabi.lib()
    m, n, k = shape
    rng = np.random.default_rng(16)
    a, b = base.dev(*base.operand(rng, m, k, pair[0], 2)), base.dev(*base.operand(rng, n, k, pair[1], 2))
    out = torch.full((m * n + 512,), 3.0, dtype=torch.bfloat16, device="cuda")
    need = L.mor_mx_matmul_workspace_bytes(m, n, k, *pair)
    assert need > 0
    ws = torch.full((need + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    _cabi.check(L.mor_mx_matmul(a[0].data_ptr(), a[1].data_ptr(), pair[0], b[0].data_ptr(), b[1].data_ptr(), pair[1], out.data_ptr(), m, n, k,
                                ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    assert (out[m * n:] == 3.0).all() and (ws[need:] == 0x5A).all()
    from mor_amd import wire
    assert torch.equal(out[: m * n].view(m, n), wire.matmul_mx(*a, *b, *pair))


@pytest.mark.parametrize("shape, pair", [((4100, 4601, 96), (A8, A8)), ((1000, 4001, 1056), (A8, C4))], ids=ids)
def test_captured_and_replayed(shape, pair):
    """The replays on changing operands, with eager calls between them, give the eager calls' bits."""
    from mor_amd import wire
    m, n, k = shape
    rng = np.random.default_rng(19)
    sets = [base.dev(*base.operand(rng, m, k, pair[0], 2), *base.operand(rng, n, k, pair[1], 2)) for _ in range(4)]
    static = [t.clone() for t in sets[0]]
    wire.matmul_mx(*static, *pair)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = wire.matmul_mx(*static, *pair)
    for i in (1, 2, 3, 0):
        for dst, src in zip(static, sets[i]):
            dst.copy_(src)
        graph.replay()
        want = wire.matmul_mx(*sets[i], *pair)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_more_small_tiles_than_2_to_the_22():
    """20 rows on 2^28 + 17 columns of 512: 69 GB of codes, 2^22 + 1 tiles of 64.  Rows of B repeat with a period, so the
    results do too; those of one period are held to the smaller product's."""
    from mor_amd import wire
    if torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved() < 120 << 30:
        pytest.skip("needs 120 GB of device memory")
    rng = np.random.default_rng(22)
    m, n, k, period = 20, 2 ** 28 + 17, 512, 4099
    (pa, sa), (pb, sb) = base.dev(*base.operand(rng, m, k, C4, 2)), base.dev(*base.operand(rng, period, k, C4, 2))
    want = wire.matmul_mx(pa, sa, pb, sb, C4)
    times = -(-n // period)
    got = wire.matmul_mx(pa, sa, pb.repeat(times, 1)[:n], sb.repeat(times, 1)[:n], C4)
    whole = n // period * period
    for r in range(m):
        assert (got[r, :whole].view(-1, period) == want[r]).all() and torch.equal(got[r, whole:], want[r, : n - whole]), r
