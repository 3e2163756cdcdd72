"""Products with weights of one's own at sizes that run by tiles of many rows: whole numbers, whose
sums fp32 holds exactly, so every output is compared bit for bit."""
import numpy as np
import pytest

import linear64 as L64
from test_gpu_linear import BackW, BackX, Forward, close, normal, stored, whole

pytestmark = pytest.mark.gpu

BF = ("bf16", "bf16", "bf16")
BF32 = ("bf16", "bf16", "f32")
# widths of one stage and less, of a few, with and without a remainder
KS = [8, 64, 72, 136, 320]


@pytest.mark.parametrize("types", [BF, BF32])
@pytest.mark.parametrize("K", KS)
@pytest.mark.parametrize("rows,n", [(1700, 1801), (2100, 4104), (129, 20500)])
def test_matmul(gpu, rows, n, K, types):
    print(f"case: k3g_matmul {rows} x {K} by {n}, {types}", flush=True)
    rng = np.random.default_rng(rows + K)
    f = Forward(rng, rows, K, n, types, "none", make=whole, bias=True, residual=True, keep=True)
    z, _, _, _, y = f.want()
    assert np.array_equal(f.got(f.z), stored(z, types[2]))
    assert np.array_equal(f.got(f.y), stored(y, types[2]))


@pytest.mark.parametrize("rows,K,n", [(1000, 72, 1500), (2100, 136, 2056), (2300, 520, 1999)])
def test_matmul_gated(gpu, rows, K, n):
    print(f"case: k3g_matmul gated {rows} x {K} by 2 x {n}", flush=True)
    rng = np.random.default_rng(rows + K)
    for types, caps in ((BF, None), (BF32, (4.0, 25.0))):
        f = Forward(rng, rows, K, n, types, "situ", keep=True, bias=True, caps=caps)
        z, z3, size, size3, y = f.want()
        close(f.got(f.z), z, L64.sum_bound(K + 2, size), types[2])
        close(f.got(f.z3), z3, L64.sum_bound(K + 2, size3), types[2])
        d, d3 = L64.sum_bound(K + 2, size), L64.sum_bound(K + 2, size3)
        close(f.got(f.y), y, 1.2 * d * (np.abs(z3) + d3) + (np.abs(z) + d) * d3 + np.abs(z * z3) * 2.0 ** -18, types[2])


# rows a token, how an expert's matrices lie (past 16 bytes), experts without one
GROUPS = [(600, 4, 1, 0, ()), (300, 6, 2, 0, (1,)), (250, 3, 3, 2, ()), (1700, 7, 1, 6, (0, 4)), (90, 5, 8, 0, ())]


@pytest.mark.parametrize("kind", ["uneven", "behind", "one"])
@pytest.mark.parametrize("K,n", [(72, 6000), (264, 2500), (8, 7001)])
@pytest.mark.parametrize("T,E,topk,skew,null", GROUPS)
def test_grouped(gpu, T, E, topk, skew, null, K, n, kind):
    print(f"case: k3g_grouped {T} x {topk} x {K} by {E} of {n}, {kind}, skew {skew}", flush=True)
    rng = np.random.default_rng(T + K + n)
    f = Forward(rng, T, K, n, BF, E=E, topk=topk, kind=kind, make=whole, skew=0, null=null, keep=True) if not skew else \
        Skewed(rng, T, K, n, E, topk, kind, skew, null)
    z, _, _, _, y = f.want()
    for e in null:
        y[f.off[e]:f.off[e + 1]] = 0
    assert np.array_equal(f.got(f.y), stored(y, "bf16"))


def Skewed(rng, T, K, n, E, topk, kind, skew, null):
    """Only the matrices lie off 16 bytes: the rows' tiles still come by DMA"""
    import test_gpu_linear as t
    table = t.table
    try:
        t.table = lambda mats, _=0: table(mats, skew)
        return Forward(rng, T, K, n, BF, E=E, topk=topk, kind=kind, make=whole, null=null, keep=True)
    finally:
        t.table = table


@pytest.mark.parametrize("types", [BF, BF32])
@pytest.mark.parametrize("rows,n,cols,E", [(1700, 64, 1808, 0), (2100, 72, 4104, 0), (1700, 200, 1800, 0), (900, 72, 3000, 5),
                                           (3000, 136, 6000, 3), (700, 8, 4000, 2)])
def test_grad_x(gpu, rows, n, cols, E, types):
    print(f"case: gradient of rows, {rows} x {n} by {cols}, {E} experts, {types}", flush=True)
    rng = np.random.default_rng(rows + n)
    for pair, add, kind in ((False, False, "uneven"), (True, True, "behind")):
        b = BackX(rng, rows, n, cols, types, E, kind, whole, pair, add)
        assert np.array_equal(b.got(b.dx), stored(b.want()[0], types[2]))


@pytest.mark.parametrize("types", [BF, BF32])
@pytest.mark.parametrize("rows,n,cols,E", [(1500, 136, 1808, 0), (2600, 72, 4000, 4)])
def test_grad_x_through_the_activation(gpu, rows, n, cols, E, types):
    print(f"case: gradient of rows through the gated activation, {rows} x {n} by {cols}, {E} experts", flush=True)
    from test_gpu_linear import slope_bound
    b = BackX(np.random.default_rng(5), rows, n, cols, types, E, "behind", normal, False, False, "situ", (4.0, 25.0))
    g, size = b.want()
    z, z3 = (v[:b.kept].astype(np.float64) for v in (b.z, b.z3))
    d, d3 = L64.slopes("situ", z, z3, *b.caps)
    own, own3 = slope_bound("situ", z, z3, d, d3)
    e = L64.sum_bound(n + 1, size)
    close(b.got(b.dx), g * d, e * np.abs(d) + (np.abs(g) + e) * own, types[2])
    close(b.got(b.dz3), g * d3, e * np.abs(d3) + (np.abs(g) + e) * own3, types[2])


@pytest.mark.parametrize("types", [BF, BF32])
@pytest.mark.parametrize("rows,n,cols,E,topk", [
    (1, 1800, 1808, 0, 1), (64, 1808, 1800, 0, 1), (65, 3000, 2904, 0, 1), (700, 1800, 1808, 0, 1),
    (400, 3000, 2904, 0, 1), (500, 520, 1032, 5, 1), (200, 1032, 1800, 4, 3), (1200, 1160, 2056, 3, 1)])
def test_grad_w(gpu, rows, n, cols, E, topk, types):
    print(f"case: gradient of matrices, {rows} x {topk}, {n} x {cols}, {E} experts, {types}", flush=True)
    rng = np.random.default_rng(rows + n + cols)
    for acc, kind in ((0, "uneven"), (1, "behind")):
        BackW(rng, rows, n, cols, types, E, topk, kind, accumulate=acc).check()


@pytest.mark.parametrize("topk", [1, 3])
def test_grad_w_rows_of_others_do_not_count(gpu, topk):
    print(f"case: gradient of matrices by tiles beside rows of NaN, topk {topk}", flush=True)
    for rows in (903, 1101):
        BackW(np.random.default_rng(rows), rows, 1032, 1800, BF32, 4, topk, "behind", poison=True, null=(2,)).check()


def test_nan_rows_stay_their_own(gpu):
    """A row of NaN or infinities among an expert's gives its own outputs only: those of the rows in the
    same tile, and of the next expert's rows, are as without it."""
    print("case: rows of NaN and infinities inside tiles", flush=True)

    def bad(rng, *shape):
        v = whole(rng, *shape)
        if shape == (900, 264):
            v[7], v[500], v[899] = np.nan, np.inf, -np.inf
        return v

    for E in (0, 4):
        f = Forward(np.random.default_rng(6), 900, 264, 4104, BF32, E=E, kind="uneven", make=bad)
        rows = np.ones(f.kept, bool)
        rows[[7, 500, 899]] = False
        f.x[[7, 500, 899]] = 0
        y = f.want()[4]
        got = f.got(f.y)
        assert np.array_equal(got[rows], stored(y, "f32")[rows])
        assert not np.isfinite(got[~rows]).all(1).any()
