"""The operators around the experts refuse what they do not take, before anything reaches a GPU
(no GPU here: a call that got as far as launching would fail too, with another message)."""
import ctypes as C

import pytest

import k3moe

F32, BF16 = k3moe.K3_WF32, k3moe.K3_WBF16
A = 0x10000                    # an address: nothing is read from it


def refused(capfd, rc, what):
    err = capfd.readouterr().err
    assert rc == -1
    assert what in err and "launch failed" not in err, err


SORT = dict(idx=A, T=4, topk=8, n_experts=64, perm=A, off=A, pos=A, err=None, work=None, work_bytes=0, stream=None)


@pytest.mark.parametrize("change,what", [
    (dict(T=-1), "tokens"), (dict(topk=0), "topk"), (dict(topk=65), "topk"), (dict(T=1 << 21), "pairs"),
    (dict(n_experts=0), "experts"), (dict(n_experts=1025), "experts"), (dict(idx=None), "missing"),
    (dict(perm=None), "missing"), (dict(off=None), "missing"), (dict(pos=None), "missing"), (dict(idx=A + 2), "aligned"),
    (dict(err=A + 1), "aligned"), (dict(T=4096), "workspace"), (dict(T=4096, work=A, work_bytes=16), "workspace"),
])
def test_sort(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_sort_tokens(*dict(SORT, **change).values()), what)


def test_sort_bytes():
    f = k3moe.lib().k3g_sort_bytes
    assert f(512, 8, 384) == 0 and f(0, 8, 384) == 0
    assert f(4096, 8, 384) > 0
    assert f(-1, 8, 384) == 0 and f(4096, 65, 384) == 0 and f(4096, 8, 1025) == 0 and f(1 << 23, 2, 8) == 0


ROWS = dict(x=A, dt=F32, T=4, topk=8, n=64, pos=A, y=A, stream=None)


@pytest.mark.parametrize("name", ["k3g_permute", "k3g_permute_grad"])
@pytest.mark.parametrize("change,what", [
    (dict(dt=2), "fp32"), (dict(T=-1), "tokens"), (dict(topk=0), "topk"), (dict(n=0), "width"),
    (dict(n=(1 << 24) + 1), "width"), (dict(x=None), "missing"), (dict(pos=None), "missing"), (dict(y=None), "missing"),
    (dict(x=A + 2), "aligned"), (dict(dt=BF16, y=A + 1), "aligned"), (dict(pos=A + 2), "aligned"),
    (dict(T=1 << 22, topk=4), "pairs"),
])
def test_rows(capfd, name, change, what):
    refused(capfd, getattr(k3moe.lib(), name)(*dict(ROWS, **change).values()), what)


UN = dict(s=A, dt=F32, T=4, topk=8, n=64, pos=A, wt=A, add=None, out=A, stream=None)


@pytest.mark.parametrize("change,what", [
    (dict(wt=None), "wt"), (dict(s=None), "missing"), (dict(out=None), "missing"), (dict(add=A + 1), "aligned"),
    (dict(dt=7), "fp32"), (dict(wt=A + 2), "aligned"), (dict(n=-5), "width"),
])
def test_unpermute(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_unpermute(*dict(UN, **change).values()), what)


GRAD = dict(dout=A, s=A, dt=BF16, T=4, topk=8, n=64, pos=A, wt=A, ds=A, dw=A, stream=None)


@pytest.mark.parametrize("change,what", [
    (dict(ds=None, dw=None), "neither"), (dict(s=None), "missing"), (dict(wt=None), "missing"),
    (dict(dout=None), "missing"), (dict(pos=None), "missing"), (dict(dw=A + 2), "aligned"), (dict(dt=-1), "fp32"),
])
def test_unpermute_grad(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_unpermute_grad(*dict(GRAD, **change).values()), what)


QUANT = dict(x=A, dt=F32, rows=4, cols=64, packed=A, scales=A, stream=None)


@pytest.mark.parametrize("change,what", [
    (dict(dt=2), "fp32"), (dict(rows=-1), "rows"), (dict(cols=48), "columns"), (dict(cols=0), "columns"),
    (dict(cols=(1 << 20) + 32), "columns"), (dict(rows=(1 << 26) + 1), "rows"), (dict(x=None), "missing"),
    (dict(x=A + 4), "aligned"), (dict(packed=None), "missing"), (dict(packed=A + 8), "aligned"),
    (dict(scales=None), "missing"),
])
def test_quant(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_quant_mxfp4(*dict(QUANT, **change).values()), what)
    d = dict(QUANT, **change)
    refused(capfd, k3moe.lib().k3g_dequant_mxfp4(d["packed"], d["scales"], d["rows"], d["cols"], d["x"], d["dt"],
                                                 None), what)


MM = dict(x=A, xdt=F32, rows=4, cols=64, w=A, n=32, y=A, ydt=F32, work=A, work_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,what", [
    (dict(xdt=2), "fp32"), (dict(ydt=9), "fp32"), (dict(cols=16), "columns"), (dict(n=8), "features"),
    (dict(n=24), "features"), (dict(n=0), "features"), (dict(w=None), "missing"), (dict(w=A + 8), "aligned"),
    (dict(y=A + 4), "aligned"), (dict(work=None), "workspace"), (dict(work_bytes=100), "workspace"),
    (dict(work=A + 8), "workspace"), (dict(rows=-3), "rows"), (dict(rows=1 << 26), "blocks"),
    (dict(rows=1 << 25, n=1 << 20, work_bytes=1 << 40), "a launch takes"),
])
def test_matmul(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_matmul_mxfp4(*dict(MM, **change).values()), what)


GR = dict(x=A, xdt=BF16, rows=4, cols=64, perm=A, topk=2, off=A, n_experts=8, w=A, w3=A, w_step=8, n=32, b1=4.0,
          b2=25.0, y=A, ydt=F32, work=A, work_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,what", [
    (dict(n_experts=0), "experts"), (dict(n_experts=1025), "experts"), (dict(topk=0), "topk"), (dict(topk=65), "topk"),
    (dict(perm=None), "topk"), (dict(off=None), "missing"), (dict(w=None), "missing"), (dict(w3=A + 4), "aligned"),
    (dict(w_step=4), "w_step"), (dict(w_step=12), "w_step"), (dict(b1=0.0), "caps"), (dict(b2=float("nan")), "caps"),
    (dict(b1=1e-35), "caps"),
    (dict(rows=1 << 22, topk=4), "pairs"), (dict(n=40), "features"), (dict(cols=100), "columns"),
    (dict(work_bytes=0), "workspace"),
])
def test_grouped(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_grouped_mxfp4(*dict(GR, **change).values()), what)


def test_work_bytes():
    f = k3moe.lib().k3g_mxfp4_work_bytes
    assert f(0, 64) == 0 and f(3, 48) == 0 and f(-1, 64) == 0
    assert f((1 << 26) - 2, 512) > 0 and f((1 << 26) - 1, 512) == 0 and f(1 << 20, 1 << 20) == 0
    assert 0 < f(1, 32) <= f(2, 32) <= f(2, 544)


def test_calls_without_rows_do_nothing():
    L = k3moe.lib()
    assert L.k3g_permute(None, F32, 0, 8, 64, None, None, None) == 0
    assert L.k3g_permute_grad(None, F32, 0, 8, 64, None, None, None) == 0
    assert L.k3g_unpermute(None, F32, 0, 8, 64, None, None, None, None, None) == 0
    assert L.k3g_unpermute_grad(None, None, F32, 0, 8, 64, None, None, A, A, None) == 0
    assert L.k3g_quant_mxfp4(None, F32, 0, 64, None, None, None) == 0
    assert L.k3g_dequant_mxfp4(None, None, 0, 64, None, F32, None) == 0
    assert L.k3g_matmul_mxfp4(None, F32, 0, 64, None, 32, None, F32, None, 0, None) == 0
    assert L.k3g_grouped_mxfp4(None, F32, 0, 64, None, 1, None, 4, None, None, 8, 32, 1.0, 1.0, None, F32, None, 0,
                               None) == 0
