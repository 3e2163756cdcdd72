"""MXFP4 products at the limits of what k3g_mxfp4_work_bytes takes."""
import ctypes as C

import numpy as np
import pytest

import k3moe
import ops64
from test_gpu_mx import bound, check, matrix, tiled

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
