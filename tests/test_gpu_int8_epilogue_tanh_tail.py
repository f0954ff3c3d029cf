"""GPU: the far tail of GELU by tanh in the epilogue of 8-bit products keeps its own size down to the smallest numbers.

Bounds, u = 2^-24, of the bias v alone (scale 0, so the product is zero). By tanh: (8 + 6 |z|) u |a|, the exponential's argument off by 6 u. Then the smallest number of the type and half a
step of it."""
import pytest
import torch

from test_gpu_int8_epilogue import BF16, F32, HALF, TINY, U, activated

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,low,high", (("gelu_tanh", -12.0, -8.0), ("gelu_tanh", -9.0, 0.0), ("gelu_tanh", -1e4, -11.0)))
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("n", (1, 8, 40, 300))
def test_tails(name, low, high, dtype, n):
    """the streaming forms and the tensor-core ones"""
    from tqllm_b200 import moe
    m, k = 4096, 64
    bank = moe.DeviceBank.from_int8(torch.ones(m, k, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda"))
    bias = torch.linspace(low, high, m)
    got = moe.linear_i8(torch.ones(n, k, dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda"), bank, out_dtype=dtype, bias=bias.cuda(), activation=name).cpu().double()
    want, own = activated(name, bias.double())
    room = U * own + HALF[dtype] * (want.abs() + U * own) + 1.5 * TINY[dtype]
    bad = ~((got - want).abs() <= room)
    assert not bool(bad.any()), f"{int(bad.sum())}: {bias.expand(n, m)[bad][:4]} {got[bad][:4]} {want.expand(n, m)[bad][:4]}"
