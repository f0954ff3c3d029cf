"""Sorted rows, their way back and the gradient of the routing weights without a GPU: the arguments that are refused before any launch."""
import pytest
import torch

from tqllm_b200 import capi, moe
from tqllm_b200.capi import lib

SHAPE, NULL, ALIGN = capi.ERR_SHAPE, capi.ERR_NULL, capi.ERR_ALIGN


def there(x=16, dt=capi.BF16, ldx=64, ids=16, plan=16, n=4, k=2, h=64, e=8, sh=0, rows=16, ldr=64, slots=16):
    return lib.b2moe_dispatch_rows(x, dt, ldx, ids, plan, n, k, h, e, sh, rows, ldr, slots, None)


def back(y=16, dt=capi.BF16, ldy=64, rows=8, slots=16, w=16, sw=None, r=None, ldr=64, n=4, k=2, h=64, sh=0, out=16, ldo=64):
    return lib.b2moe_combine_rows(y, dt, ldy, rows, slots, w, sw, r, ldr, n, k, h, sh, out, ldo, None)


def back_grad(g=16, dt=capi.BF16, ldg=64, y=16, ldy=64, rows=8, slots=16, w=16, sw=None, n=4, k=2, h=64, sh=0, gy=16, ldgy=64, gw=16, gs=None):
    return lib.b2moe_combine_rows_backward(g, dt, ldg, y, ldy, rows, slots, w, sw, n, k, h, sh, gy, ldgy, gw, gs, None)


def route(gating=1, l=16, ld=8, ids=16, w=16, g=16, sw=None, gs=None, e=8, k=2, norm=1, scale=1.0, n=4, out=16, ldo=8, add=0):
    return lib.b2moe_route_backward(gating, l, ld, ids, w, g, sw, gs, e, k, norm, scale, n, out, ldo, add, None)


def each(f, status, cases):
    assert [f(**c) for c in cases] == [status] * len(cases)


def test_there():
    each(there, SHAPE, (dict(n=0), dict(n=-3), dict(k=0), dict(n=1 << 29, k=2), dict(h=0), dict(h=60, ldx=64), dict(h=66, ldx=72, dt=capi.F32), dict(dt=4), dict(e=0), dict(sh=-1), dict(sh=5), dict(ldx=56), dict(ldx=68), dict(ldr=56),
                        dict(ldr=66, dt=capi.F32)))
    each(there, NULL, (dict(x=None), dict(ids=None), dict(plan=None), dict(rows=None)))
    each(there, ALIGN, (dict(x=24), dict(rows=8), dict(ids=18), dict(plan=18), dict(slots=18)))


def test_back():
    each(back, SHAPE, (dict(n=0), dict(k=0), dict(n=1 << 29, k=2), dict(h=0), dict(h=60), dict(dt=-1), dict(rows=0), dict(sh=3), dict(ldy=56), dict(ldy=68), dict(r=16, ldr=56), dict(ldo=0), dict(ldo=68)))
    each(back, NULL, (dict(y=None), dict(slots=None), dict(out=None)))
    each(back, ALIGN, (dict(y=24), dict(r=24), dict(out=24), dict(slots=18), dict(w=18), dict(sw=18)))


def test_back_gradient():
    each(back_grad, SHAPE, (dict(n=0), dict(k=0), dict(h=60), dict(dt=9), dict(rows=0), dict(sh=2), dict(gs=16), dict(ldg=56), dict(ldy=68), dict(ldgy=56)))
    each(back_grad, NULL, (dict(g=None), dict(slots=None), dict(gy=None, gw=None), dict(y=None)))
    each(back_grad, ALIGN, (dict(g=24), dict(y=24), dict(gy=24), dict(slots=18), dict(w=18), dict(sw=18), dict(gw=18), dict(gs=18, sh=4)))


def test_route_gradient():
    each(route, SHAPE, (dict(gating=0), dict(gating=3), dict(e=0), dict(e=4097, ldo=5000), dict(k=0), dict(k=9), dict(n=0), dict(ldo=7), dict(sw=16, gs=16), dict(gating=2, ld=7), dict(scale=float("inf")), dict(scale=float("nan"))))
    each(route, NULL, (dict(ids=None), dict(w=None), dict(g=None), dict(out=None), dict(gating=2, l=None), dict(gs=16, ldo=9)))
    each(route, ALIGN, (dict(ids=18), dict(w=18), dict(g=18), dict(out=18), dict(l=18), dict(sw=18), dict(sw=16, gs=18, ldo=9)))


def refused(status, f, **k):
    with pytest.raises(capi.B2moeError) as e:
        f(**k)
    assert e.value.status == status


def test_python():
    t, i32 = torch.zeros, torch.int32
    plan = moe.Plan(8, 4, 2, 0, "cpu")
    for bad in (dict(x=t(3, 64)), dict(x=t(4, 64).double()), dict(x=t(64, 4).t()), dict(ids=t(4, 2)), dict(ids=t(3, 2, dtype=i32)), dict(ids=t(4, 3, dtype=i32)), dict(ids=t(2, 4, dtype=i32).t()), dict(rows=t(7, 64)),
                dict(rows=t(8, 64).half()), dict(rows=t(8, 60))):
        refused(SHAPE, moe.dispatch_rows, **{**dict(x=t(4, 64), ids=t(4, 2, dtype=i32), plan=plan), **bad})
    refused(capi.ERR_CUDA, moe.dispatch_rows, x=t(4, 64), ids=t(4, 2, dtype=i32), plan=plan)
    good = dict(y=t(8, 64), slots=t(8, dtype=i32), weights=t(4, 2), n=4, topk=2)
    for bad in (dict(y=t(8, 64).double()), dict(y=t(64, 8).t()), dict(slots=t(8)), dict(slots=t(9, dtype=i32)), dict(slots=t(16, dtype=i32)[::2]), dict(weights=t(4, 3)), dict(weights=t(4, 2).double()), dict(weights=t(2, 4).t()),
                dict(shared_weights=t(4)), dict(slots=t(12, dtype=i32), shared_weights=t(5)), dict(residual=t(4, 60)), dict(residual=t(4, 64).half()), dict(out=t(3, 64)), dict(out=t(64, 4).t())):
        refused(SHAPE, moe.combine_rows, **{**good, **bad})
    refused(capi.ERR_CUDA, moe.combine_rows, **good)
    good["grad_out"] = t(4, 64)
    for bad in (dict(grad_out=t(4, 60)), dict(grad_out=t(4, 64).half()), dict(grad_y=t(7, 64)), dict(grad_y=t(64, 8).t()), dict(shared_weights=t(4)), dict(weights=t(8).double())):
        refused(SHAPE, moe.combine_rows_backward, **{**good, **bad})
    refused(capi.ERR_CUDA, moe.combine_rows_backward, **good)
    good = dict(logits=t(4, 8), ids=t(4, 2, dtype=i32), weights=t(4, 2), grad_weights=t(4, 2), experts=8)
    for bad in (dict(logits=t(4, 7)), dict(logits=t(3, 8)), dict(logits=t(4, 8).double()), dict(logits=t(8, 4).t()), dict(ids=t(4, 2)), dict(ids=t(2, 4, dtype=i32).t()), dict(weights=t(4, 3)), dict(grad_weights=t(4, 2).double()),
                dict(weights=t(2, 4).t()), dict(shared_weights=t(4)), dict(grad_shared=t(4)), dict(shared_weights=t(4), grad_shared=t(3)), dict(out=t(4, 7)), dict(out=t(4, 8), shared_weights=t(4), grad_shared=t(4)), dict(out=t(8, 4).t()),
                dict(out=t(4, 8).double())):
        refused(SHAPE, moe.route_backward, **{**good, **bad})
    refused(capi.ERR_CUDA, moe.route_backward, **good)
