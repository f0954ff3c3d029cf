"""Tensors of the wrong kind are refused by the Python mirror before any call (CPU tensors: nothing would be launched)."""
import pytest
import torch

from tqllm_b200 import capi, moe


def refused(status, f, *a, **k):
    with pytest.raises(capi.B2moeError) as e:
        f(*a, **k)
    assert e.value.status == status


def test_banks():
    w, v = torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6)
    assert (moe.DeviceBank.from_int8(w, v, 2).experts, moe.DeviceBank.from_int8(w.view(3, 2, 32), v.view(3, 2)).rows) == (2, 2)
    for bad in ((w.float(), v, 1), (w, v.double(), 1), (w.t(), v, 1), (torch.zeros(6, 64, dtype=torch.int8)[:, :32], v, 1)):
        refused(capi.ERR_FORMAT, moe.DeviceBank.from_int8, *bad)
    for bad in ((w, v[:5], 1), (w, v, 4)):
        refused(capi.ERR_SHAPE, moe.DeviceBank.from_int8, *bad)


def test_rows_and_products():
    refused(capi.ERR_SHAPE, moe.quantize_rows, torch.zeros(32, 4).t())
    q, s, bank = torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4), moe.DeviceBank.from_int8(torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6))
    for bad in ((q.float(), s), (q[:, :16], s), (q, s[:3]), (q, s.double()), (q, torch.zeros(8)[::2]), (torch.zeros(32, 4, dtype=torch.int8).t(), s)):
        refused(capi.ERR_SHAPE, moe.linear_i8, *bad, bank)
    for out in (torch.zeros(4, 5), torch.zeros(3, 6), torch.zeros(6, 4).t()):
        refused(capi.ERR_SHAPE, moe.linear_i8, q, s, bank, out=out)
    for status in (torch.zeros(1), torch.zeros(4, dtype=torch.uint8), torch.zeros(0, dtype=torch.int32)):
        refused(capi.ERR_SHAPE, lambda: moe.linear_i8(q, s, bank, status=status))


def test_balance():
    l, ids = torch.zeros(5, 8), torch.zeros(5, 2, dtype=torch.int32)
    for bad in (dict(logits=l.double()), dict(logits=l[:, :7]), dict(logits=torch.zeros(8, 5).t()), dict(ids=ids.long()), dict(ids=ids[:4]), dict(ids=torch.zeros(2, 5, dtype=torch.int32).t()),
                dict(mask=torch.ones(4, dtype=torch.bool)), dict(mask=torch.ones(5)), dict(offsets=torch.tensor([0, 5])), dict(offsets=torch.tensor([0], dtype=torch.int32))):
        refused(capi.ERR_SHAPE, moe.balance_loss, **{**dict(logits=l, ids=ids, experts=8, coef=0.1), **bad})
    saved = moe.Balance(torch.zeros(()), torch.zeros(1, 8, dtype=torch.int32), torch.zeros(1, 8), torch.zeros(2, dtype=torch.int32))
    for bad in (dict(offsets=torch.tensor([0, 2, 5], dtype=torch.int32)), dict(grad_loss=torch.zeros((), dtype=torch.float64)), dict(out=torch.zeros(5, 7)), dict(out=torch.zeros(4, 8)),
                dict(out=torch.zeros(5, 8, dtype=torch.float64)), dict(out=torch.zeros(8, 5).t()), dict(logits=l[:, :7])):
        refused(capi.ERR_SHAPE, moe.balance_loss_backward, **{**dict(logits=l, saved=saved, topk=2, coef=0.1), **bad})


def test_what_the_balance_gradient_is_given():
    """counts as they come back from a reduction over ranks, say"""
    l, f = torch.zeros(5, 8), torch.zeros(())
    counts, tokens = torch.zeros(1, 8, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for c, t, g in ((counts.long(), tokens, None), (counts.float(), tokens, None), (torch.zeros(1, 16, dtype=torch.int32)[:, ::2], tokens, None),
                    (counts, tokens.long(), None), (counts, tokens[:1], None), (counts, torch.zeros(4, dtype=torch.int32)[::2], None), (counts, tokens, torch.zeros(0)), (counts, tokens, torch.zeros(2))):
        refused(capi.ERR_SHAPE, moe.balance_loss_backward, l, moe.Balance(f, c, f, t), 2, 0.1, grad_loss=g)


def test_tensors_that_are_not_on_the_current_device():
    x, q, s = torch.zeros(4, 32), torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4)
    bank = moe.DeviceBank.from_int8(torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6))
    l, ids = torch.zeros(5, 8), torch.zeros(5, 2, dtype=torch.int32)
    saved = moe.Balance(torch.zeros(()), torch.zeros(1, 8, dtype=torch.int32), torch.zeros(1, 8), torch.zeros(2, dtype=torch.int32))
    refused(capi.ERR_CUDA, moe.quantize_rows, x)
    refused(capi.ERR_CUDA, moe.linear_i8, q, s, bank)
    refused(capi.ERR_CUDA, moe.balance_loss, l, ids, 8, 0.1)
    refused(capi.ERR_CUDA, moe.balance_loss_backward, l, saved, 2, 0.1)
