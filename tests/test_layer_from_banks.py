"""MoeLayer.from_banks looks at what it is given beside the banks: a router of another type or size than the kernels read is refused (CPU tensors: nothing would be launched)."""
import pytest
import torch

from tqllm_b200 import capi, moe, synth


def bank(experts, rows, cols):
    return moe.DeviceBank.from_int8(torch.zeros(experts, rows, cols, dtype=torch.int8), torch.zeros(experts, rows))


def test_what_lies_beside_the_banks():
    shape = synth.LayerShape("beside", 64, 4, 2, 32)
    banks = [bank(4, 32, 64), bank(4, 32, 64), bank(4, 64, 32)]
    f = lambda router=torch.zeros(4, 64), **k: moe.MoeLayer.from_banks(shape, router, banks, **k)
    for bad in (dict(router=torch.zeros(4, 64).bfloat16()), dict(router=torch.zeros(4, 64).half()), dict(router=torch.zeros(3, 64)), dict(router=torch.zeros(4, 32)), dict(router=torch.zeros(64, 4).t()),
                dict(router=torch.zeros(4, 128)[:, :64]), dict(router=torch.zeros(256)), dict(sel_bias=torch.zeros(3)), dict(sel_bias=torch.zeros(4).double()), dict(sel_bias=torch.zeros(8)[::2]),
                dict(shared_gate_vec=torch.zeros(32)), dict(shared_gate_vec=torch.zeros(64).bfloat16()), dict(shared_gate_vec=torch.zeros(1, 64))):
        with pytest.raises(capi.B2moeError) as e:
            f(**bad)
        assert e.value.status == capi.ERR_SHAPE
    with pytest.raises(capi.B2moeError) as e:                          # what is right so far is looked at for where it lies
        f(sel_bias=torch.zeros(4), shared_gate_vec=torch.zeros(64))
    assert e.value.status == capi.ERR_CUDA
