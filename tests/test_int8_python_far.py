"""Sizes and strides that the C ABI holds in 32 bits are refused beyond them by the Python mirror, instead of being taken by their low bits (tensors without memory)."""
import pytest
import torch

from tqllm_b200 import capi, moe

FAR = 1 << 32
meta = lambda shape, stride, dtype: torch.empty_strided(shape, stride, dtype=dtype, device="meta")


def refused(f, *a, **k):
    with pytest.raises(capi.B2moeError) as e:
        f(*a, **k)
    assert e.value.status == capi.ERR_SHAPE


def test_rows_and_products():
    refused(moe.quantize_rows, meta((2, FAR + 16), (FAR + 16, 1), torch.bfloat16))
    refused(moe.quantize_rows, meta((FAR + 2, 16), (16, 1), torch.bfloat16))
    refused(moe.DeviceBank.from_int8, meta((1, FAR + 16), (FAR + 16, 1), torch.int8), meta((1,), (1,), torch.float32))
    refused(moe.DeviceBank.from_int8, meta((FAR + 2, 16), (16, 1), torch.int8), meta((FAR + 2,), (1,), torch.float32))
    refused(moe.DeviceBank.from_int8, meta((FAR + 1, 1, 16), (16, 16, 1), torch.int8), meta((FAR + 1, 1), (1, 1), torch.float32))
    bank = moe.DeviceBank.from_int8(torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6))
    refused(moe.linear_i8, meta((FAR + 4, 32), (32, 1), torch.int8), meta((FAR + 4,), (1,), torch.float32), bank)


def test_balance():
    l, ids = torch.zeros(5, 8), torch.zeros(5, 2, dtype=torch.int32)
    saved = moe.Balance(torch.zeros(()), torch.zeros(1, 8, dtype=torch.int32), torch.zeros(1, 8), torch.zeros(2, dtype=torch.int32))
    far = meta((5, 8), (FAR + 8, 1), torch.float32)
    refused(moe.balance_loss, far, ids, 8, 0.1)
    refused(moe.balance_loss_backward, far, saved, 2, 0.1)
    refused(moe.balance_loss_backward, l, saved, 2, 0.1, out=far)
    refused(moe.balance_loss, meta((FAR + 5, 8), (8, 1), torch.float32), meta((FAR + 5, 2), (2, 1), torch.int32), 8, 0.1)
    refused(moe.balance_loss, l, ids, 8, 0.1, offsets=meta((FAR + 3,), (1,), torch.int32))
    one = meta((1, 8), (FAR + 8, 1), torch.float32)                    # one row: its stride is not looked at
    with pytest.raises(capi.B2moeError) as e:
        moe.balance_loss(one, ids[:1], 8, 0.1)
    assert e.value.status == capi.ERR_CUDA
