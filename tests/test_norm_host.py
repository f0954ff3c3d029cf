"""The norm and its gradient without a GPU: the arguments that are refused before any launch, and the workspace's size."""
import pytest
import torch

from tqllm_b200 import capi, moe
from tqllm_b200.capi import lib

SHAPE, NULL, ALIGN, WORKSPACE = capi.ERR_SHAPE, capi.ERR_NULL, capi.ERR_ALIGN, capi.ERR_WORKSPACE
NAN, INF = float("nan"), float("inf")


def norm(x=16, dt=capi.BF16, ldx=64, r=16, ldr=64, w=16, wdt=capi.F32, eps=1e-6, n=2, k=64, s=16, lds=64, y=16, ldy=64, q=16, ldq=64, scale=16):
    return lib.b2moe_rms_norm(x, dt, ldx, r, ldr, w, wdt, eps, n, k, s, lds, y, ldy, q, ldq, scale, None)


def test_norm_refusals():
    bad = (dict(n=0), dict(n=-1), dict(n=1 << 30), dict(k=0), dict(k=16400, ldx=16400, ldr=16400, lds=16400, ldy=16400, ldq=16400), dict(dt=3), dict(wdt=capi.F16), dict(wdt=7), dict(eps=-1.0), dict(eps=NAN),
           dict(eps=INF), dict(ldx=63), dict(ldx=0), dict(ldr=56), dict(lds=56), dict(ldy=56), dict(ldq=48), dict(ldq=72), dict(k=56), dict(k=8))
    assert [norm(**b) for b in bad] == [SHAPE] * len(bad)
    bad = (dict(x=None), dict(w=None), dict(y=None, q=None), dict(scale=None), dict(r=None))
    assert [norm(**b) for b in bad] == [NULL] * len(bad)
    bad = (dict(x=17), dict(r=17), dict(s=17), dict(y=17), dict(w=18), dict(q=24), dict(scale=18), dict(x=24), dict(r=24), dict(s=24), dict(y=24), dict(w=24), dict(ldx=68), dict(ldr=66))
    assert [norm(**b) for b in bad] == [ALIGN] * len(bad)


def grad(h=16, dt=capi.BF16, ldh=64, w=16, wdt=capi.F32, g=16, ldg=64, s=16, lds=64, eps=1e-6, n=2, k=64, dx=16, ldx=64, dw=16, acc=0, ws=16, size=1 << 20):
    return lib.b2moe_rms_norm_backward(h, dt, ldh, w, wdt, g, ldg, s, lds, eps, n, k, dx, ldx, dw, acc, ws, size, None)


def test_gradient_refusals():
    bad = (dict(n=0), dict(n=1 << 30), dict(k=0), dict(k=16385, ldh=16385, ldg=16385, lds=16385, ldx=16385), dict(dt=3), dict(wdt=capi.F16), dict(eps=-1.0), dict(eps=NAN), dict(ldh=63), dict(ldg=63), dict(lds=63), dict(ldx=63))
    assert [grad(**b) for b in bad] == [SHAPE] * len(bad)
    bad = (dict(h=None), dict(w=None), dict(g=None), dict(dx=None), dict(ws=None))
    assert [grad(**b) for b in bad] == [NULL] * len(bad)
    bad = (dict(h=17), dict(w=18), dict(g=17), dict(s=17), dict(dx=17), dict(dw=18), dict(ws=24))
    assert [grad(**b) for b in bad] == [ALIGN] * len(bad)
    need = lib.b2moe_rms_norm_backward_workspace_bytes(2, 64)
    assert need >= 2 * 64 * 4 and grad(size=need - 1) == WORKSPACE


def test_workspace_grows():
    for k in (1, 100, 2048, 4096, 16384):
        sizes = [lib.b2moe_rms_norm_backward_workspace_bytes(n, k) for n in (1, 2, 100, 147, 148, 149, 295, 296, 297, 5000, (1 << 30) - 1)]
        assert sizes == sorted(sizes) and sizes[0] >= 4 * k and sizes[-1] <= 40 << 20
    assert [lib.b2moe_rms_norm_backward_workspace_bytes(*a) for a in ((0, 8), (1 << 30, 8), (8, 0), (8, 16385))] == [0] * 4


def refused(status, f, *a, **k):
    with pytest.raises(capi.B2moeError) as e:
        f(*a, **k)
    assert e.value.status == status


def test_python_refusals():
    x, w, t = torch.zeros(4, 32), torch.zeros(32), torch.zeros
    for bad in (dict(x=x.double()), dict(x=t(128)), dict(x=t(32, 4).t()), dict(weight=w[:31]), dict(weight=w.half()), dict(weight=t(64)[::2]), dict(residual=x[:3]), dict(residual=x.half()), dict(residual=t(32, 4).t()),
                dict(sum_out=x), dict(residual=x, sum_out=t(4, 31)), dict(out=t(4, 33)), dict(out=x.bfloat16()), dict(out=x, rows=False, quantize=True)):
        refused(SHAPE, moe.rms_norm, **{**dict(x=x, weight=w, eps=1e-6), **bad})
    for bad in (dict(h=x.double()), dict(weight=w.half()), dict(grad_y=x.half()), dict(grad_y=x[:2]), dict(grad_sum=t(4, 31)), dict(out=t(32, 4).t()), dict(grad_weight=w.double()), dict(grad_weight=w[:3]),
                dict(grad_weight=t(64)[::2]), dict(grad_weight=w, weight_grad=False)):
        refused(SHAPE, moe.rms_norm_backward, **{**dict(h=x, weight=w, grad_y=x, eps=1e-6), **bad})
    refused(capi.ERR_CUDA, moe.rms_norm, x, w, 1e-6)
    refused(capi.ERR_CUDA, moe.rms_norm_backward, x, w, x, 1e-6)
