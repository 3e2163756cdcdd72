"""MXFP4 products long enough for each kernel's steady state: at least four quads of 512 columns, so
that the loads of the next quad run beside the products of this one in every tile and for every wave
that shares the columns; outputs of more than 256 MB, whose stores are streamed; and the same of the
values' own quantisation. Against plain 64-bit forms."""
import ctypes as C

import numpy as np
import pytest

import k3moe
import ops64
import test_gpu_mx as small
from test_gpu_order import DT

pytestmark = pytest.mark.gpu


# from 1056 columns on a wave alone has three quads; waves that share the columns by eights and fours
# loop from 4608 and 2560 on. 4128, 3616, 4640, 1632, 1696 and 1760 columns end inside a quad, and
# inside one of its four chunks. In order: the columns shared by 8 waves with 1, by 4 with 2 and 4 row
# blocks of 16 places, by 4 of 32 and of 64 places, then a wave's own columns: 64 places by 192 and
# 256 features, 128 by 192 and 256.
@pytest.mark.parametrize("rows,cols,n", [(3, 4640, 80), (16, 4640, 80), (64, 4640, 1648), (300, 4128, 640),
                                         (257, 3616, 1616), (600, 4128, 1040), (400, 1632, 6144), (512, 1696, 7152),
                                         (1000, 1632, 6096), (2000, 1760, 7088)])
@pytest.mark.parametrize("xdt,ydt", [("f32", "f32"), ("bf16", "bf16")])
def test_matmul(gpu, rows, cols, n, xdt, ydt):
    small.test_matmul(gpu, rows, cols, n, xdt, ydt)


# a few tokens that meet an expert about once (quantised in the kernel); 16 and 32 places; 64 and 128
@pytest.mark.parametrize("T,k,E,cols,n,drop", [(12, 4, 40, 4640, 96, 0.0), (16, 2, 33, 4128, 64, 0.2),
                                               (100, 4, 40, 4640, 96, 0.1), (200, 4, 24, 4128, 112, 0.1),
                                               (300, 4, 40, 1760, 1648, 0.1)])
@pytest.mark.parametrize("kind", ["tokens", "gated", "situ", "rows"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_grouped(gpu, T, k, E, cols, n, drop, kind, dt):
    small.test_grouped(gpu, T, k, E, cols, n, drop, kind, dt)


@pytest.mark.parametrize("kind", ["tokens", "situ"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_grouped_128_places(gpu, kind, dt):
    small.test_grouped(gpu, 1500, 2, 8, 1760, 2832, 0.0, kind, dt)


def matrices(rng, E, n, cols):
    """E tiled matrices, the table of their addresses, and their values on the GPU in 64 bits"""
    import torch
    made = small.experts(rng, E, cols, n, 1, 120, 123)[0]
    return made[0], torch.from_numpy(made[1].astype(np.int64)).cuda(), [torch.from_numpy(v).cuda() for v in made[2]]


def quantised(x, period):
    """The 64-bit values of x's rows in MXFP4, x's first `period` rows repeating"""
    import torch
    v = ops64.values(*ops64.quant(x[:period].float().cpu().numpy()))
    return torch.from_numpy(v).cuda()


def close(got, want, mag, cols, eps):
    """bound() of test_gpu_mx, and the output's rounding"""
    tol = (cols // 32 + 16) * 2.0 ** -23 * mag
    bad = (got.double() - want).abs() > tol + eps * (want.abs() + tol) * (1 + 2.0 ** -7)
    assert not bool(bad.any()), (bad.nonzero()[:4], got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("rows,cols,n,ydt", [(20000, 160, 3600, "f32"), (40000, 160, 3600, "bf16"),
                                             (384000, 160, 192, "f32")])
def test_streamed_outputs(gpu, rows, cols, n, ydt):
    """One matrix, an output of more than 256 MB: every row."""
    import torch
    print(f"case: k3g_matmul_mxfp4 {rows} x {cols} by {n}, streamed {ydt}", flush=True)
    L = k3moe.lib()
    tag, _, eps = DT[ydt]
    t = torch.bfloat16 if ydt == "bf16" else torch.float32
    assert rows * n * (2 if ydt == "bf16" else 4) > 1 << 28
    period = 1000
    x = torch.randn(period, cols, device="cuda").repeat(rows // period, 1).contiguous()
    bufs, tab, (w,) = matrices(np.random.default_rng(n), 1, n, cols)
    y = torch.empty(rows, n, dtype=t, device="cuda")
    size = L.k3g_mxfp4_work_bytes(rows, cols)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert L.k3g_matmul_mxfp4(x.data_ptr(), k3moe.K3_WF32, rows, cols, C.c_void_p(bufs[0].ptr), n, y.data_ptr(), tag,
                              work.data_ptr(), size, None) == 0
    torch.cuda.synchronize()
    xv = quantised(x, period)
    want, mag = xv @ w.T, xv.abs() @ w.abs().T
    for r in range(0, rows, period):
        close(y[r:r + period], want, mag, cols, eps)


@pytest.mark.parametrize("ydt", ["f32", "bf16"])
def test_streamed_outputs_of_gated_experts(gpu, ydt):
    """Gate and up of sorted rows, an output of more than 256 MB; rows behind the last place stay."""
    import torch
    rows, cols, n, E = 40000, 160, 3600, 4
    print(f"case: k3g_grouped_mxfp4 {rows} x {cols} by {n}, gated, streamed {ydt}", flush=True)
    L = k3moe.lib()
    tag, _, eps = DT[ydt]
    t = torch.bfloat16 if ydt == "bf16" else torch.float32
    period = 1000
    # gates of a few units: 160 products of weights of about 2^-5 and values of about 1
    x = torch.randn(period, cols, device="cuda").repeat(rows // period, 1).contiguous()
    rng = np.random.default_rng(3)
    b1, tab1, w1 = matrices(rng, E, n, cols)
    b3, tab3, w3 = matrices(rng, E, n, cols)
    off = torch.tensor([0, 9000, 9000, 30500, 39001], dtype=torch.int32, device="cuda")
    y = torch.full((rows, n), 7.0, dtype=t, device="cuda")
    size = L.k3g_mxfp4_work_bytes(rows, cols)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert L.k3g_grouped_mxfp4(x.data_ptr(), k3moe.K3_WF32, rows, cols, None, 1, off.data_ptr(), E, tab1.data_ptr(),
                               tab3.data_ptr(), 8, n, 4.0, 25.0, y.data_ptr(), tag, work.data_ptr(), size, None) == 0
    torch.cuda.synchronize()
    xv = quantised(x, period)
    for e, (a, b) in enumerate(((0, 9000), (9000, 9000), (9000, 30500), (30500, 39001))):
        g, u = xv @ w1[e].T, xv @ w3[e].T
        tg, tu = ((cols // 32 + 16) * 2.0 ** -23 * (xv.abs() @ w[e].abs().T) for w in (w1, w3))
        want = 4.0 * torch.tanh(g / 4.0) * torch.sigmoid(g) * 25.0 * torch.tanh(u / 25.0)
        # as test_gpu_mx: |d act / d gate| <= 1.25 |up|, |act| <= |gate| |up|, the activation itself 2^-19
        tol = 1.25 * tg * (u.abs() + tu) + g.abs() * tu + 2.0 ** -19 * want.abs()
        for r in range(a, b, period):
            # row r + i repeats row (r + i) % period
            first = r % period
            m = min(period, b - r)
            at = (torch.arange(m, device="cuda") + first) % period
            v = want[at]
            bad = (y[r:r + m].double() - v).abs() > tol[at] + eps * (v.abs() + tol[at]) * (1 + 2.0 ** -7)
            assert not bool(bad.any()), (e, r, bad.nonzero()[:4])
    assert bool((y[39001:] == 7.0).all())


def test_streamed_values(gpu):
    """More than 256 MB of fp32 values to MXFP4 and back: every block."""
    import torch
    rows, cols, period = 20000, 3616, 400
    print(f"case: k3g_quant_mxfp4 and k3g_dequant_mxfp4 {rows} x {cols}, fp32", flush=True)
    assert rows * cols * 4 > 1 << 28
    L = k3moe.lib()
    first = small.spread(np.random.default_rng(8), period, cols)
    x = torch.from_numpy(first).cuda().repeat(rows // period, 1).contiguous()
    pk = torch.empty(rows, cols // 2, dtype=torch.uint8, device="cuda")
    sc = torch.empty(rows, cols // 32, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert L.k3g_quant_mxfp4(x.data_ptr(), 0, rows, cols, pk.data_ptr(), sc.data_ptr(), None) == 0
    torch.cuda.synchronize()
    code, scale = ops64.quant(first)
    assert torch.equal(pk, torch.from_numpy(ops64.pack(code)).cuda().repeat(rows // period, 1))
    assert torch.equal(sc, torch.from_numpy(scale).cuda().repeat(rows // period, 1))
    x.zero_()
    torch.cuda.synchronize()
    assert L.k3g_dequant_mxfp4(pk.data_ptr(), sc.data_ptr(), rows, cols, x.data_ptr(), 0, None) == 0
    torch.cuda.synchronize()
    want = torch.from_numpy(ops64.values(code, scale)).float().cuda().repeat(rows // period, 1)
    assert torch.equal(x, want)
