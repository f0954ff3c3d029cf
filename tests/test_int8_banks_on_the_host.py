"""A bank over arrays that lie in host memory (a checkpoint as it was loaded) and calls that would launch on it: refused by the Python mirror before the library is reached, whose kernels would read
host addresses. CPU tensors only: nothing is launched."""
import types

import pytest
import torch

from tqllm_b200 import capi, moe, synth


class Reached(AssertionError):
    pass


@pytest.fixture
def no_launch(monkeypatch):
    """the library without what launches: sizes and views stay"""
    def reached(name):
        def call(*a):
            raise Reached(name)
        return call
    names = ("b2moe_expert_gateup_swiglu", "b2moe_expert_down", "b2moe_dequant_dump", "b2moe_layer_forward", "b2moe_layer_forward_residual")
    stand_in = types.SimpleNamespace(**{n: getattr(capi.lib, n) for n in capi.SIGNATURES if n not in names}, **{n: reached(n) for n in names})
    monkeypatch.setattr(moe, "lib", stand_in)
    monkeypatch.setattr(moe, "_stream", lambda: 0)                     # what a machine with a GPU has


def bank(experts, rows, cols):
    return moe.DeviceBank.from_int8(torch.zeros(experts, rows, cols, dtype=torch.int8), torch.zeros(experts, rows))


def refused(f, *a, **k):
    with pytest.raises(capi.B2moeError) as e:
        f(*a, **k)
    assert e.value.status == capi.ERR_CUDA and "current CUDA device" in str(e.value)


def test_expert_products(no_launch):
    plan = moe.Plan(4, 3, 2, 0, "cpu")
    refused(moe.expert_gateup_swiglu, bank(4, 32, 64), bank(4, 32, 64), torch.zeros(3, 64), plan)
    refused(moe.expert_gateup_swiglu, bank(4, 32, 64), bank(4, 32, 64), torch.zeros(3, 64), plan, act=torch.zeros(6, 32))
    refused(moe.expert_down, bank(4, 64, 32), torch.zeros(6, 32), plan)
    refused(moe.expert_down, bank(4, 64, 32), torch.zeros(6, 32), plan, y=torch.zeros(6, 64))


def test_dump(no_launch):
    refused(bank(2, 16, 32).dequant)


def test_layers(no_launch):
    shape = synth.LayerShape("host", 64, 4, 2, 32)
    refused(moe.MoeLayer.from_banks, shape, torch.zeros(4, 64), [bank(4, 32, 64), bank(4, 32, 64), bank(4, 64, 32)])
    layer = moe.MoeLayer.__new__(moe.MoeLayer)
    layer.router_w = torch.zeros(4, 64)
    refused(layer.forward, torch.zeros(3, 64))
