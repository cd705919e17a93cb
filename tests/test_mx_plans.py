"""Which kernels a product of MX tensors takes, without a GPU."""
import ctypes as C

import pytest

import mx_plain as P
from mor_amd import _cabi

L = _cabi.lib()
FORMATS = (P.E4M3, P.E5M2, P.E2M1)
PAIRS = [(a, b) for a in FORMATS for b in FORMATS]


def plan(m, n, k, a_fmt, b_fmt):
    out = (C.c_int64 * 8)()
    _cabi.check(L.mor_mx_matmul_plan(m, n, k, a_fmt, b_fmt, out))
    return dict(zip(("tile", "waves", "parts", "rows", "cols", "rest_tile", "rest_waves", "threads"), out))


def test_refusals():
    out = (C.c_int64 * 8)()
    assert L.mor_mx_matmul_plan(8, 8, 64, 0, 0, None) == -1 and b"NULL" in L.mor_last_error()
    for shape in ((0, 8, 64, 0, 0), (8, 8, 48, 0, 0), (8, 1 << 30, 64, 0, 0), (8, 8, 64, 2, 0), (8, 8, 64, 0, 3)):
        assert L.mor_mx_matmul_plan(*shape, out) == -1 and b"no such product" in L.mor_last_error()


@pytest.mark.parametrize("pair", PAIRS, ids=str)
def test_no_launch_has_2_to_the_32_threads(pair):
    """A grid of 2^32 threads is cut without an error.  16 columns a workgroup of four waves reach that 15 columns before
    2^28, one row of 64 x 64 tiles 63 columns before 2^30."""
    near = [(1 << e) + d for e in (26, 27, 28, 29) for d in (-64, -17, -16, -15, -1, 0, 1, 17)] + [(1 << 30) - d for d in (129, 128, 127, 65, 64, 63, 1)]
    for long in near:
        for short in (1, 2, 16, 17, 32):
            for k in (32, 512, 544, 1536, 1568, 2080, 8192, (1 << 23) - 32):
                for m, n in ((short, long), (long, short)):
                    if m * n <= 1 << 35:
                        assert plan(m, n, k, *pair)["threads"] < 1 << 32, (m, n, k)
    for m, n in ((129, 266000000), (266000000, 129), (1 << 17, 1 << 18), (4097, 8000000), (200, 170000000)):
        assert plan(m, n, 32, *pair)["threads"] < 1 << 32, (m, n)


def test_the_few_row_kernel_ends_where_its_grid_does():
    at = lambda n: plan(1, n, 1568, P.E2M1, P.E2M1)  # noqa: E731
    assert at((1 << 28) - 16)["tile"] == 0 and at((1 << 28) - 16)["waves"] == 4
    for n in ((1 << 28) - 15, (1 << 28) - 1, 1 << 28):
        assert at(n)["tile"] != 0


def kind(shape, pair):
    """the kernels and launches of a product: widths of the codes, tile, waves, k split or not, what is cut, the rest's tiles"""
    q = plan(*shape, *pair)
    cut = "rows" if q["rows"] < shape[0] else "columns" if q["cols"] < shape[1] else ""
    return ("4x4" if pair == (P.E2M1, P.E2M1) else "8x4" if P.E2M1 in pair else "8x8", q["tile"], q["waves"], q["parts"] > 1, cut, q["rest_tile"], q["rest_waves"])


def test_every_kind_of_plan_is_among_the_tested_sizes():
    """Plans of sizes drawn over the whole range, against those of the sizes that the GPU tests multiply exactly."""
    import random
    import test_gpu_mx_matmul as base
    import test_gpu_mx_plans as more
    # (the largest sizes of the older list run with three of the pairs)
    few = ((P.E4M3, P.E4M3), (P.E2M1, P.E2M1), (P.E4M3, P.E2M1))
    tested = {kind(s, p) for s in base.SHAPES for p in base.PAIRS if p in few or s[0] * s[1] <= 1 << 20} | {kind(s, p) for s, p in more.CASES}
    rng = random.Random(20)
    size = lambda top: round(2 ** rng.uniform(0, top))  # noqa: E731
    drawn = {}
    for _ in range(40000):
        shape, pair = (size(16.1), size(16.1), 32 * size(9.3)), rng.choice(few)
        drawn.setdefault(kind(shape, pair), shape)
    missing = {k: s for k, s in drawn.items() if k not in tested}
    assert len(drawn) > 40 and not missing, missing
