"""MXFP4 products at the limits: of what k3g_mxfp4_work_bytes takes, and of what numbers are."""
import ctypes as C

import numpy as np
import pytest

import k3moe
import ops64
from test_gpu_mx import bound, check, experts, grouped, matrix, tiled
from test_gpu_order import Out, dev, routing

pytestmark = pytest.mark.gpu


def test_most_activation_blocks(gpu):
    """2^26 - 1 blocks of 512 columns with the row of zeros, the most there may be: a wave each
    would be 2^32 threads, which is more than a launch has. The rows repeat, so every one of them
    is compared with the first, and those with the 64-bit form."""
    import torch
    L = k3moe.lib()
    rows, cols, n, period = (1 << 26) - 2, 32, 16, 1202
    assert rows % period == 0
    size = L.k3g_mxfp4_work_bytes(rows, cols)
    assert size == (rows + 1) * 272 and L.k3g_mxfp4_work_bytes(rows + 1, cols) == 0
    print(f"case: k3g_matmul_mxfp4 {rows} x {cols} by {n}, bf16", flush=True)
    rng = np.random.default_rng(1)
    pk, sc, w = matrix(rng, n, cols)
    t = tiled(pk, sc, n, cols)
    first = torch.randn(period, cols, device="cuda").bfloat16()
    x = first.unsqueeze(0).expand(rows // period, period, cols).contiguous()
    y = torch.full((rows // period, period, n), 7.0, dtype=torch.bfloat16, device="cuda")
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert L.k3g_matmul_mxfp4(x.data_ptr(), k3moe.K3_WBF16, rows, cols, C.c_void_p(t.ptr), n, y.data_ptr(),
                              k3moe.K3_WBF16, work.data_ptr(), size, None) == 0
    torch.cuda.synchronize()
    xv = ops64.values(*ops64.quant(first.float().cpu().numpy()))
    check(y[0].float().cpu().numpy().astype(np.float64), xv @ w.T, bound(xv, w)[1], "bf16")
    assert bool((y == y[0]).all())


@pytest.mark.parametrize("rows,n", [(3, 64), (40, 64), (500, 6144)])
def test_infinities_by_zeros(gpu, rows, n):
    """A row with an infinity or a NaN is NaN by weights of zero too."""
    print(f"case: k3g_matmul_mxfp4 with infinities by zeros, {rows} rows", flush=True)
    cols = 1056
    x = np.random.default_rng(rows).normal(0, 1, (rows, cols)).astype(np.float32)
    x[1, 700], x[rows - 1, 1055] = np.inf, np.nan
    t = tiled(np.zeros((n, cols // 2), np.uint8), np.full((n, cols // 32), 127, np.uint8), n, cols)
    L = k3moe.lib()
    b, p = dev(x)
    size = L.k3g_mxfp4_work_bytes(rows, cols)
    work, y = Out(np.uint8, size), Out(np.float32, rows * n)
    assert L.k3g_matmul_mxfp4(p, 0, rows, cols, C.c_void_p(t.ptr), n, y.ptr, 0, work.ptr, size, None) == 0
    k3moe.sync()
    got = y.get().reshape(rows, n)
    bad = np.zeros(rows, bool)
    bad[[1, rows - 1]] = True
    assert np.isnan(got[bad]).all() and (got[~bad] == 0).all()


@pytest.mark.parametrize("T,E,n", [(5, 4, 32), (200, 4, 32), (400, 4, 1648)])
@pytest.mark.parametrize("caps", [(2.0 ** 100, 2.0 ** 100), (4.0, 25.0)])
def test_infinities_through_the_activation(gpu, T, E, n, caps):
    """The same of a gated product, whichever of the experts the row meets; other rows are numbers."""
    print(f"case: k3g_grouped_mxfp4 with infinities, {T} tokens, caps {caps}", flush=True)
    rng = np.random.default_rng(T)
    k, cols = 2, 1056
    idx = routing(rng, T, k, E)
    perm, off, _ = ops64.order(idx, E)
    x = rng.normal(0, 1, (T, cols)).astype(np.float32)
    x[1, 700], x[T - 1, 5] = -np.inf, np.nan
    mats = experts(rng, E, cols, n, 2, 120, 123)
    got = grouped(x, "f32", perm, k, off, [m[1] for m in mats], n, "f32", T * k, caps)
    bad = np.isin(perm // k, (1, T - 1))
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
