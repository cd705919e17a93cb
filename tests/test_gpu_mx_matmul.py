"""The product of two tensors in the MX wire format (wire.matmul_mx) against float64."""
import numpy as np
import pytest
import torch

import mx_plain as P

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

FORMATS = (P.E4M3, P.E5M2, P.E2M1)
PAIRS = [(a, b) for a in FORMATS for b in FORMATS]
NAMES = {P.E4M3: "E4M3", P.E5M2: "E5M2", P.E2M1: "E2M1"}
# (m, n, k): one row, one column, one block; every kernel and both sides of each choice between them; sizes that end inside
# tiles, steps and groups; k that is a multiple of 512, 128, 64 and 32; k split over workgroups
SHAPES = [(1, 1, 32), (1, 16, 96), (3, 50, 512), (16, 33, 544), (17, 1000, 2080), (32, 4100, 1024), (33, 1, 64), (64, 130, 4096),
          (65, 33, 32), (100, 129, 160), (128, 128, 4096), (129, 257, 4160), (197, 1031, 1056), (513, 256, 14336), (1100, 1000, 320),
          (600, 4001, 352), (1100, 4008, 160), (61, 33000, 96), (33000, 120, 64),
          (700, 1000, 14336), (3585, 3333, 96), (3840, 3328, 1056), (3584, 3600, 2048), (4096, 3584, 1664)]


def ids(v):
    return "x".join(NAMES.get(x, str(x)) if len(v) == 2 else str(x) for x in v)


def operand(rng, rows, k, fmt, spread):
    """codes over the whole format (no NaNs), scales within `spread` binary orders, as (payload, scales) on the host"""
    top = len(P.table(fmt))
    codes = rng.integers(0, top, (rows, k)) | (rng.integers(0, 2, (rows, k)) << (P.BITS[fmt] - 1))
    scales = rng.integers(127 - spread, 128 + spread, (rows, k // 32)).astype(np.uint8)
    return P.pack(codes.astype(np.uint8), fmt), scales


def dev(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


def run(a, b, fmts):
    from mor_amd import wire
    return wire.matmul_mx(*dev(*a), *dev(*b), *fmts)


@pytest.mark.parametrize("pair", PAIRS, ids=ids)
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_one_code_per_row_gives_exact_products(shape, pair):
    """Each row of a has one non-zero code, so a result is one product of two codes and two scales: exact in bf16 (two
    significands of at most 4 bits).  Every column of k, every scale byte and every place of the output is met exactly."""
    m, n, k = shape
    if pair not in ((P.E4M3, P.E4M3), (P.E2M1, P.E2M1), (P.E4M3, P.E2M1)) and m * n > 1 << 20:
        pytest.skip("the large shapes run with three of the nine pairs")
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    (pa, sa), (pb, sb) = operand(rng, m, k, pair[0], 20), operand(rng, n, k, pair[1], 20)
    at = (np.arange(m) * 37 + rng.integers(0, 5)) % k
    ca = P.unpack(pa, pair[0])
    keep = np.zeros_like(ca)
    keep[np.arange(m), at] = ca[np.arange(m), at]
    pa = P.pack(keep, pair[0])
    va, vb = P.decode(pa, sa, pair[0]), P.decode(pb, sb, pair[1])
    want = va[np.arange(m), at][:, None] * vb[:, at].T
    got = P.to64(run((pa, sa), (pb, sb), pair))
    assert np.array_equal(got, want), np.argwhere(got != want)[:4]


@pytest.mark.parametrize("pair", PAIRS, ids=ids)
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] * s[1] * s[2] < 1 << 28], ids=ids)
def test_full_rows(shape, pair):
    m, n, k = shape
    rng = np.random.default_rng(m + n + k)
    a, b = operand(rng, m, k, pair[0], 3), operand(rng, n, k, pair[1], 3)
    want, bound = P.product_bound(P.decode(*a, pair[0]), P.decode(*b, pair[1]), exact_products=pair == (P.E2M1, P.E2M1))
    got = P.to64(run(a, b, pair))
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)


@pytest.mark.parametrize("shape", [(1, 64, 8192), (128, 192, 14336), (3584, 3600, 2048)], ids=ids)
def test_four_bit_products_lose_nothing_but_the_sums_roundings(shape):
    """Codes of E2M1 and one scale: the products are multiples of 1/4 up to 36, whose sums are exact in fp32, so that the
    result is the exact sum rounded once."""
    m, n, k = shape
    rng = np.random.default_rng(k)
    (pa, sa), (pb, sb) = operand(rng, m, k, P.E2M1, 1), operand(rng, n, k, P.E2M1, 1)
    sa[:], sb[:] = 127, 125
    va, vb = torch.from_numpy(P.decode(pa, sa, P.E2M1)).cuda(), torch.from_numpy(P.decode(pb, sb, P.E2M1)).cuda()
    want = (va @ vb.t()).to(torch.bfloat16)                       # exact in float64
    assert torch.equal(run((pa, sa), (pb, sb), (P.E2M1, P.E2M1)), want)


@pytest.mark.parametrize("shape", [(5, 40, 96), (40, 40, 96), (130, 140, 1056), (3585, 3333, 96)], ids=ids)
def test_nans_stay_in_their_row_and_column(shape):
    m, n, k = shape
    rng = np.random.default_rng(5)
    (pa, sa), (pb, sb) = operand(rng, m, k, P.E4M3, 2), operand(rng, n, k, P.E2M1, 2)
    sa[m - 1, -1] = 255                      # the E8M0 NaN, in the last row and block
    pa[2, 0] = 0x7F                          # a NaN code
    sb[n - 2, 0] = 255
    nan = np.zeros((m, n), bool)
    nan[[2, m - 1]] = True
    nan[:, n - 2] = True
    got = P.to64(run((pa, sa), (pb, sb), (P.E4M3, P.E2M1)))
    assert np.array_equal(np.isnan(got), nan)
    va, vb = P.decode(pa, sa, P.E4M3), P.decode(pb, sb, P.E2M1)
    want, bound = P.product_bound(np.nan_to_num(va), np.nan_to_num(vb))
    assert (np.abs(got - want) <= bound)[~nan].all()


@pytest.mark.parametrize("shape", [(1, 1, 32), (17, 33, 96), (65, 33, 32), (130, 139, 544), (100, 64, 14336), (3585, 3333, 96)], ids=ids)
def test_nothing_behind_the_output_is_written(shape):
    from mor_amd import _cabi
    L = _cabi.lib()
    m, n, k = shape
    rng = np.random.default_rng(6)
    a, b = dev(*operand(rng, m, k, P.E2M1, 2)), dev(*operand(rng, n, k, P.E2M1, 2))
    out = torch.full((m * n + 512,), 3.0, dtype=torch.bfloat16, device="cuda")
    need = L.mor_mx_matmul_workspace_bytes(m, n, k, 4, 4)
    ws = torch.full((need + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    _cabi.check(L.mor_mx_matmul(a[0].data_ptr(), a[1].data_ptr(), 4, b[0].data_ptr(), b[1].data_ptr(), 4, out.data_ptr(), m, n, k,
                                ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    assert (out[m * n:] == 3.0).all() and (ws[need:] == 0x5A).all()
    from mor_amd import wire
    assert torch.equal(out[: m * n].view(m, n), wire.matmul_mx(*a, *b, wire.E2M1))


def test_zero_sizes():
    from mor_amd import wire
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")  # noqa: E731
    assert wire.matmul_mx(u8(0, 64), u8(0, 2), u8(5, 64), u8(5, 2)).shape == (0, 5)
    assert wire.matmul_mx(u8(3, 64), u8(3, 2), u8(0, 64), u8(0, 2)).shape == (3, 0)
    empty = wire.matmul_mx(u8(3, 0), u8(3, 0), u8(4, 0), u8(4, 0))
    assert empty.shape == (3, 4) and (empty == 0).all()


def test_views_of_the_operands():
    """Rows cut out of larger operands (scales that begin at any byte) and a column range (copied) give the same bits."""
    from mor_amd import wire
    rng = np.random.default_rng(8)
    for m, n, k in ((20, 300, 1056), (200, 300, 1056)):
        (pa, sa), (pb, sb) = dev(*operand(rng, m + 3, k, P.E4M3, 2)), dev(*operand(rng, n + 1, k, P.E2M1, 2))
        got = wire.matmul_mx(pa[3:], sa[3:], pb[1:], sb[1:], wire.E4M3, wire.E2M1)
        want = wire.matmul_mx(pa[3:].clone(), sa[3:].clone(), pb[1:].clone(), sb[1:].clone(), wire.E4M3, wire.E2M1)
        assert torch.equal(got, want)
        cut = wire.matmul_mx(pa[:, 64:128], sa[:, 2:4], pb[:, 32:64], sb[:, 2:4], wire.E4M3, wire.E2M1)
        assert torch.equal(cut, wire.matmul_mx(pa[:, 64:128].contiguous(), sa[:, 2:4].contiguous(), pb[:, 32:64].contiguous(),
                                               sb[:, 2:4].contiguous(), wire.E4M3, wire.E2M1))


@pytest.mark.parametrize("shape", [(4, 512, 4096), (100, 64, 14336), (3584, 3584, 512)], ids=ids)
def test_captured_and_replayed(shape):
    """Two graphs of different products, replayed in turn on changing operands, with eager calls between them: each replay
    gives the eager call's bits."""
    from mor_amd import wire
    m, n, k = shape
    rng = np.random.default_rng(9)
    sets = [dev(*operand(rng, m, k, P.E4M3, 2), *operand(rng, n, k, P.E4M3, 2)) for _ in range(4)]
    static = [[t.clone() for t in sets[0]] for _ in range(2)]
    wire.matmul_mx(*static[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(wire.matmul_mx(*s))
        graphs.append(g)
    for i in range(4):
        which = i % 2
        for dst, src in zip(static[which], sets[i]):
            dst.copy_(src)
        graphs[which].replay()
        graphs[1 - which].replay()
        want = wire.matmul_mx(*sets[i])
        torch.cuda.synchronize()
        assert torch.equal(outs[which], want), i


def test_more_columns_than_the_few_row_kernel_has_threads_for():
    """2^28 + 17 rows of B: offsets and a grid past 32 bits.  Rows of B repeat with a period, so the results do too."""
    from mor_amd import wire
    rng = np.random.default_rng(12)
    n, period = 2 ** 28 + 17, 4099
    (pa, sa), (pb, sb) = dev(*operand(rng, 1, 32, P.E2M1, 2)), dev(*operand(rng, period, 32, P.E2M1, 2))
    times = -(-n // period)
    got = wire.matmul_mx(pa, sa, pb.repeat(times, 1)[:n], sb.repeat(times, 1)[:n], wire.E2M1)
    want = wire.matmul_mx(pa, sa, pb, sb, wire.E2M1)
    whole = n // period * period
    assert got.shape == (1, n) and (got[0, :whole].view(-1, period) == want).all() and torch.equal(got[0, whole:], want[0, : n - whole])


def test_two_streams_at_once():
    from mor_amd import wire
    rng = np.random.default_rng(10)
    work = [dev(*operand(rng, 300, 14336, P.E2M1, 2), *operand(rng, 200, 14336, P.E2M1, 2)) for _ in range(2)]
    want = [wire.matmul_mx(*w, wire.E2M1) for w in work]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(wire.matmul_mx(*work[i], wire.E2M1))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.parametrize("rows", [(300000, 40), (40, 300000)], ids=ids)
def test_operands_and_outputs_past_32_bit_offsets(rows):
    """2.4 GB of codes on either side; sampled rows and columns against float64."""
    from mor_amd import wire
    m, n = rows
    k = 8192
    g = torch.Generator(device="cuda").manual_seed(3)
    codes = lambda r: torch.randint(0, 0x70, (r, k), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
    scales = lambda r: torch.randint(120, 130, (r, k // 32), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
    pa, sa, pb, sb = codes(m), scales(m), codes(n), scales(n)
    got = wire.matmul_mx(pa, sa, pb, sb)
    at_a, at_b = [torch.tensor(sorted({0, 1, r // 2, r - 2, r - 1})) for r in (m, n)]
    side = lambda p, s, at: P.decode(p[at.cuda()].cpu().numpy(), s[at.cuda()].cpu().numpy(), P.E4M3)  # noqa: E731
    want, bound = P.product_bound(side(pa, sa, at_a), side(pb, sb, at_b))
    assert (np.abs(P.to64(got[at_a.cuda()][:, at_b.cuda()]) - want) <= bound).all()
