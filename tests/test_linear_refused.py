"""The products with weights of one's own refuse what they do not take, before anything reaches a
GPU (no GPU here: a call that got as far as launching would fail too, with another message)."""
import ctypes as C

import pytest

import k3moe
from test_ops_refused import A, BF16, F32, refused


def epilogue(**f):
    ep = k3moe.K3gEpilogue()
    for k, v in f.items():
        setattr(ep, k, v)
    return C.byref(ep)


def back(**f):
    b = k3moe.K3gBack()
    for k, v in f.items():
        setattr(b, k, v)
    return C.byref(b)


SITU = dict(act=k3moe.K3G_ACT_SITU, b1=4.0, b2=25.0)
MM = dict(x=A, xdt=F32, rows=4, cols=65, w=A, w3=None, wdt=F32, n=33, ep=None, y=A, ydt=F32, stream=None)
GR = dict(x=A, xdt=F32, rows=4, cols=65, perm=A, topk=2, off=A, E=8, w=A, w3=None, step=8, wdt=F32, n=33, ep=None, y=A,
          ydt=F32, stream=None)
FORWARD = [
    (dict(xdt=2), "x is fp32"), (dict(wdt=3), "w is fp32"), (dict(ydt=-1), "y is fp32"), (dict(rows=-1), "rows"),
    (dict(rows=(1 << 23) + 1), "rows"), (dict(cols=0), "columns"), (dict(cols=(1 << 20) + 1), "columns"),
    (dict(n=0), "features"), (dict(n=(1 << 20) + 1), "features"), (dict(x=None), "missing"), (dict(w=None), "missing"),
    (dict(y=None), "missing"), (dict(x=A + 2), "aligned"), (dict(y=A + 2), "aligned"),
    (dict(xdt=BF16, x=A + 1), "aligned"), (dict(w3=A), "two products"), (dict(ep=epilogue(**SITU)), "two products"),
    (dict(ep=epilogue(act=6)), "no activation"), (dict(ep=epilogue(act=-1)), "no activation"),
    (dict(w3=A, ep=epilogue(act=k3moe.K3G_ACT_SITU, b1=1.0)), "caps"),
    (dict(w3=A, ep=epilogue(act=k3moe.K3G_ACT_SITU, b1=float("nan"), b2=1.0)), "caps"),
    (dict(ep=epilogue(bias=A + 2)), "bias"), (dict(ep=epilogue(bias3=A)), "second matrix"),
    (dict(ep=epilogue(z3=A)), "second matrix"), (dict(ep=epilogue(residual=A + 2)), "residual"),
    (dict(ep=epilogue(z=A + 1)), "z is missing or not"), (dict(rows=1 << 23, n=1 << 20, topk=1), "a launch takes"),
]


@pytest.mark.parametrize("change,what", FORWARD + [(dict(w=A + 2), "aligned")])
def test_matmul(capfd, change, what):
    change = {k: v for k, v in change.items() if k != "topk"}
    refused(capfd, k3moe.lib().k3g_matmul(*dict(MM, **change).values()), what)


@pytest.mark.parametrize("change,what", FORWARD + [
    (dict(E=0), "experts"), (dict(E=1025), "experts"), (dict(topk=0), "topk"), (dict(topk=65), "topk"),
    (dict(perm=None), "topk"), (dict(perm=A + 2), "aligned"), (dict(off=None), "missing"), (dict(off=A + 1), "aligned"),
    (dict(step=4), "w_step"), (dict(step=12), "w_step"), (dict(w=A + 4), "aligned"), (dict(rows=1 << 22, topk=4), "pairs"),
])
def test_grouped(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_grouped(*dict(GR, **change).values()), what)


GX = dict(dy=A, dy3=None, dydt=BF16, rows=4, n=33, w=A, w3=None, wdt=F32, cols=65, back=None, dx=A, dxdt=F32,
          stream=None)
BACK = [
    (dict(dydt=2), "dy is fp32"), (dict(wdt=2), "w is fp32"), (dict(dxdt=2), "dx is fp32"), (dict(rows=-1), "rows"),
    (dict(n=0), "features"), (dict(cols=0), "columns"), (dict(dy=None), "missing"), (dict(w=None), "missing"),
    (dict(dx=None), "missing"), (dict(dy=A + 1), "aligned"), (dict(dx=A + 2), "aligned"), (dict(dy3=A), "together"),
    (dict(w3=A), "together"), (dict(back=back(add=A + 2)), "add"), (dict(back=back(act=1)), "z is missing"),
    (dict(back=back(act=7, z=A)), "no activation"), (dict(back=back(z=A, z3=A, act=5, b1=1.0, b2=1.0)), "dz3"),
    (dict(back=back(z3=A, dz3=A, act=5, b1=1.0, b2=1.0)), "belong"), (dict(back=back(z=A, act=5, b1=1.0, b2=1.0)), "two"),
    (dict(back=back(z=A, z3=A, dz3=A, act=2)), "two"), (dict(back=back(z=A, z3=A, dz3=A, act=5)), "caps"),
    (dict(back=back(z=A + 2, act=1)), "z is missing or not"),
]


@pytest.mark.parametrize("change,what", BACK)
def test_grad_x(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_matmul_grad_x(*dict(GX, **change).values()), what)
    d = dict(GX, **change)
    refused(capfd, k3moe.lib().k3g_grouped_grad_x(d["dy"], d["dy3"], d["dydt"], d["rows"], d["n"], A, 8, d["w"],
                                                  d["w3"], 8, d["wdt"], d["cols"], d["back"], d["dx"], d["dxdt"],
                                                  None), what)


GXG = dict(dy=A, dy3=None, dydt=BF16, rows=4, n=33, off=A, E=8, w=A, w3=None, step=8, wdt=F32, cols=65, back=None, dx=A,
           dxdt=F32, stream=None)


@pytest.mark.parametrize("change,what", [(dict(off=None), "missing"), (dict(E=0), "experts"), (dict(step=9), "w_step"),
                                         (dict(w=A + 2), "aligned"), (dict(rows=1 << 24), "rows")])
def test_grouped_grad_x(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_grouped_grad_x(*dict(GXG, **change).values()), what)


GW = dict(dy=A, dydt=BF16, x=A, xdt=F32, rows=4, n=33, cols=65, accumulate=0, dw=A, dwdt=F32, db=None, stream=None)
GWG = dict(dy=A, dydt=BF16, x=A, xdt=F32, rows=4, n=33, cols=65, perm=A, topk=2, off=A, E=8, accumulate=0, dw=A, step=8,
           dwdt=F32, db=None, stream=None)
WEIGHTS = [
    (dict(dydt=2), "dy is fp32"), (dict(xdt=2), "x is fp32"), (dict(dwdt=2), "dw is fp32"), (dict(rows=-1), "rows"),
    (dict(n=0), "features"), (dict(cols=0), "columns"), (dict(dy=None), "missing"), (dict(x=None), "missing"),
    (dict(dw=None), "missing"), (dict(dw=A + 2), "aligned"), (dict(dy=A + 1), "aligned"), (dict(db=A + 2), "dbias"),
]


@pytest.mark.parametrize("change,what", WEIGHTS)
def test_grad_w(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_matmul_grad_w(*dict(GW, **change).values()), what)


@pytest.mark.parametrize("change,what", WEIGHTS + [
    (dict(off=None), "missing"), (dict(off=None, rows=0), "missing"), (dict(E=0), "experts"), (dict(perm=None), "topk"),
    (dict(topk=65), "topk"), (dict(step=12), "dw_step"), (dict(dw=A + 4), "aligned"),
    (dict(n=1 << 20, cols=1 << 20, E=1024), "a launch takes"),
])
def test_grouped_grad_w(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_grouped_grad_w(*dict(GWG, **change).values()), what)


AG = dict(dh=A, dt=F32, rows=4, n=33, act=2, b1=0.0, b2=0.0, z=A, z3=None, dz=A, dz3=None, stream=None)


@pytest.mark.parametrize("change,what", [
    (dict(dt=2), "dh is fp32"), (dict(rows=-1), "rows"), (dict(n=0), "values"), (dict(n=(1 << 24) + 1), "values"),
    (dict(rows=(1 << 26) + 1), "rows"), (dict(act=9), "no activation"), (dict(dh=None), "missing"),
    (dict(z=None), "missing"), (dict(dz=None), "missing"), (dict(z3=A), "gated"), (dict(dz3=A), "gated"),
    (dict(act=5, z3=A, dz3=A + 4), "caps"), (dict(act=5, b1=1.0, b2=1.0), "missing"),
    (dict(act=5, b1=1.0, b2=1.0, z3=A, dz3=A), "the same"), (dict(z=A + 2), "aligned"),
])
def test_act_grad(capfd, change, what):
    refused(capfd, k3moe.lib().k3g_act_grad(*dict(AG, **change).values()), what)


def test_calls_without_rows_do_nothing():
    L = k3moe.lib()
    assert L.k3g_matmul(None, F32, 0, 64, None, None, F32, 32, None, None, F32, None) == 0
    assert L.k3g_matmul_grad_x(None, None, F32, 0, 32, None, None, F32, 64, None, None, F32, None) == 0
    assert L.k3g_matmul_grad_w(None, F32, None, F32, 0, 32, 64, 1, A, F32, None, None) == 0
    assert L.k3g_grouped(None, F32, 0, 64, None, 1, None, 8, None, None, 8, F32, 32, None, None, F32, None) == 0
    assert L.k3g_grouped_grad_x(None, None, F32, 0, 32, None, 8, None, None, 8, F32, 64, None, None, F32, None) == 0
    assert L.k3g_grouped_grad_w(None, F32, None, F32, 0, 32, 64, None, 1, A, 8, 1, A, 8, F32, None, None) == 0
    assert L.k3g_act_grad(None, F32, 0, 8, 2, 0.0, 0.0, None, None, None, None, None) == 0
