"""8-bit products with an epilogue without a GPU: the arguments that are refused before any launch."""
import ctypes as C

import pytest
import torch

from tqllm_b200 import capi, moe
from tqllm_b200.capi import lib


def bank(experts=1, rows=32, cols=256, data=16, aux=16, kind=capi.I8):
    return capi.Bank(data, aux, kind, experts, rows, cols)


def call(w=bank(), q=16, ldq=256, s=16, n=2, b=16, act=1, r=16, ldr=32, y=16, dt=capi.BF16, ldy=32):
    return lib.b2moe_linear_i8_epilogue(q, ldq, s, C.byref(w), n, b, act, r, ldr, y, dt, ldy, None, None)


def test_refusals():
    each = lambda status, cases: [call(**c) for c in cases] == [status] * len(cases)
    assert each(capi.ERR_SHAPE, (dict(act=-1), dict(act=5), dict(ldr=31), dict(ldr=0), dict(n=0), dict(dt=5), dict(ldq=240), dict(ldy=31), dict(w=bank(2)), dict(w=bank(cols=250))))
    assert each(capi.ERR_NULL, (dict(q=None), dict(s=None), dict(y=None), dict(w=bank(data=None))))
    assert each(capi.ERR_ALIGN, (dict(b=18), dict(r=17), dict(r=18, dt=capi.F32), dict(q=8), dict(y=17)))
    assert call(w=bank(kind=12)) == capi.ERR_FORMAT


def test_python():
    t = torch.zeros
    q, s, w = t(4, 32, dtype=torch.int8), t(4), moe.DeviceBank.from_int8(t(6, 32, dtype=torch.int8), t(6))
    for bad in (dict(activation="tanh"), dict(activation=None), dict(activation=3), dict(bias=t(5)), dict(bias=t(6).half()), dict(bias=t(12)[::2]), dict(residual=t(4, 6)), dict(residual=t(4, 5).bfloat16()), dict(residual=t(3, 6).bfloat16()),
                dict(residual=t(6, 4).bfloat16().t()), dict(out=t(4, 6), residual=t(4, 6).bfloat16())):
        with pytest.raises(capi.B2moeError) as e:
            moe.linear_i8(q, s, w, **bad)
        assert e.value.status == capi.ERR_SHAPE
    for good in (dict(activation="gelu"), dict(bias=t(6)), dict(residual=t(4, 6).bfloat16()), dict(out=t(4, 6), residual=t(4, 6))):
        with pytest.raises(capi.B2moeError) as e:
            moe.linear_i8(q, s, w, **good)
        assert e.value.status == capi.ERR_CUDA
