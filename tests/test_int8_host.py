"""8-bit banks and the balance loss without a GPU: sizes, and the arguments that are refused before any launch."""
import ctypes as C

import pytest

from tqllm_b200 import capi
from tqllm_b200.capi import lib

I8 = capi.I8


def bank(experts=4, rows=32, cols=256, data=16, aux=16):
    return capi.Bank(data, aux, I8, experts, rows, cols)


def test_sizes():
    assert lib.b2moe_bank_bytes(I8, 19, 48) == 19 * 48 and lib.b2moe_bank_aux_bytes(I8, 19, 48) == 19 * 4
    assert lib.b2moe_bank_bytes(I8, 19, 40) == 0 and lib.b2moe_bank_bytes(I8, 1, 1 << 17) == 0 and lib.b2moe_bank_bytes(I8, 1, (1 << 17) - 16) == (1 << 17) - 16
    assert lib.b2moe_raw_bytes(I8, 16, 256) == 0
    assert lib.b2moe_bank_load(I8, 16, 1, 16, 256, 16, 16, None) == capi.ERR_FORMAT
    assert lib.b2moe_expert_workspace_bytes(I8, 7, 48, capi.BF16) >= 7 * (48 + 4) and lib.b2moe_expert_workspace_bytes(I8, 7, 40, capi.BF16) == 0
    sizes = [lib.b2moe_expert_slot_workspace_bytes(C.byref(bank()), n, capi.F32) for n in range(1, 3000, 7)]
    assert sizes == sorted(sizes) and all(lib.b2moe_expert_workspace_bytes(I8, n, 256, capi.F32) <= s for n, s in zip(range(1, 3000, 7), sizes))
    for e in (1, 32, 33, 512, 4096):
        for seqs in (1, 7, 65535):
            sizes = [lib.b2moe_balance_workspace_bytes(e, n, seqs) for n in (1, 7, 8, 9, 2367, 2368, 2369, 37887, 37888, 37889, 1 << 20, 1 << 22)]
            assert sizes == sorted(sizes) and sizes[0] > 0
    assert lib.b2moe_balance_workspace_bytes(4097, 8, 1) == 0 and lib.b2moe_balance_workspace_bytes(8, 0, 1) == 0 and lib.b2moe_balance_workspace_bytes(8, 8, 65536) == 0


def test_layer_workspace_of_8_bit_banks():
    L = capi.Layer(hidden=1024, experts=64, topk=6, ff=528, has_shared=1)
    L.gate = L.up = bank(64, 528, 1024)
    L.down = bank(64, 1024, 528)
    before = 0
    for n in range(1, 700, 3):
        v = capi.LayerWs()
        assert lib.b2moe_layer_workspace(C.byref(L), n, C.byref(v)) == 0
        assert v.total >= before and v.total - v.expert_scratch >= n * 7 * (528 + 4)
        before = v.total


def test_quantize_refusals():
    f = lambda x=16, dt=capi.BF16, ldx=64, n=2, k=64, q=16, ldq=64, s=16: lib.b2moe_quantize_rows(x, dt, ldx, n, k, q, ldq, s, None)
    assert [f(n=0), f(k=0), f(k=24), f(k=1 << 17, ldx=1 << 17, ldq=1 << 17), f(dt=3), f(ldx=56), f(ldx=68), f(ldq=48), f(ldq=72)] == [capi.ERR_SHAPE] * 9
    assert f(ldx=66, dt=capi.F32) == capi.ERR_SHAPE
    assert [f(x=None), f(q=None), f(s=None)] == [capi.ERR_NULL] * 3
    assert [f(x=24), f(q=8), f(s=18)] == [capi.ERR_ALIGN] * 3


def test_linear_refusals():
    f = lambda w, q=16, ldq=256, s=16, n=2, y=16, dt=capi.BF16, ldy=32: lib.b2moe_linear_i8(q, ldq, s, C.byref(w), n, y, dt, ldy, None, None)
    one = bank(1)
    assert [f(bank(2)), f(one, n=0), f(one, dt=5), f(one, ldq=240), f(one, ldq=264), f(one, ldy=31), f(bank(1, cols=250)), f(bank(1, rows=0))] == [capi.ERR_SHAPE] * 8
    assert [f(one, q=None), f(one, s=None), f(one, y=None), f(bank(1, data=None)), f(bank(1, aux=None))] == [capi.ERR_NULL] * 5
    assert [f(one, q=8), f(bank(1, data=24)), f(one, y=17), f(one, y=18, dt=capi.F32), f(one, s=18), f(bank(1, aux=18))] == [capi.ERR_ALIGN] * 6
    assert f(capi.Bank(16, None, 12, 1, 32, 256)) == capi.ERR_FORMAT
    assert lib.b2moe_linear_i8(16, 256, 16, None, 2, 16, 0, 32, None, None) == capi.ERR_NULL


def test_product_refusals():
    b, q4 = bank(), capi.Bank(16, None, 12, 4, 32, 256)
    gateup = lambda g, u, ws=None, size=0, act=16: lib.b2moe_expert_gateup_swiglu(C.byref(g), C.byref(u), None, None, 16, capi.BF16, 16, 2, 2, 0, act, ws, size, None)
    assert gateup(b, q4) == capi.ERR_FORMAT and gateup(b, bank(rows=48)) == capi.ERR_SHAPE and gateup(b, bank(aux=None)) == capi.ERR_NULL
    assert gateup(b, b) == capi.ERR_NULL and gateup(b, b, 16, 100) == capi.ERR_WORKSPACE and gateup(b, b, 24, 1 << 20) == capi.ERR_ALIGN
    down = lambda ws, size: lib.b2moe_expert_down(C.byref(b), None, 16, 16, 2, 2, 0, 16, ws, size, None)
    assert down(None, 0) == capi.ERR_NULL and down(16, 4 * 260 - 1) == capi.ERR_WORKSPACE
    # the library's own array is checked like any other scratch: rows that do not fit are refused
    assert lib.b2moe_expert_down_static(C.byref(bank(4, 32, 1 << 16)), None, 16, 16, 300, 2, 0, 16, None) == capi.ERR_CAPACITY


def test_balance_refusals():
    def loss(gating=1, logits=16, ld=8, ids=16, topk=2, mask=None, offsets=16, seqs=2, experts=8, n=4, out=16, counts=16, prob=16, tokens=16, ws=16, size=1 << 20):
        return lib.b2moe_balance_loss(gating, logits, ld, ids, topk, mask, offsets, seqs, experts, n, 0.1, out, counts, prob, tokens, ws, size, None)
    bad = [loss(gating=0), loss(gating=3), loss(ld=7), loss(topk=0), loss(topk=9), loss(offsets=None), loss(seqs=0), loss(seqs=65536), loss(experts=0), loss(n=0),
           loss(experts=4097, ld=5000), loss(n=1 << 30, topk=2)]
    assert bad == [capi.ERR_SHAPE] * len(bad)
    null = [loss(**{k: None}) for k in ("logits", "ids", "out", "counts", "prob", "tokens", "ws")]
    assert null == [capi.ERR_NULL] * len(null)
    assert [loss(ws=24), loss(logits=18), loss(ids=18), loss(offsets=18), loss(counts=17), loss(prob=18), loss(tokens=18), loss(out=18)] == [capi.ERR_ALIGN] * 8
    assert loss(size=lib.b2moe_balance_workspace_bytes(8, 4, 2) - 1) == capi.ERR_WORKSPACE

    def back(gating=1, logits=16, ld=8, topk=2, offsets=16, seqs=2, experts=8, n=4, counts=16, tokens=16, grad=16, ldg=8):
        return lib.b2moe_balance_loss_backward(gating, logits, ld, topk, None, offsets, seqs, experts, n, 0.1, counts, tokens, None, grad, ldg, 0, None)
    bad = [back(gating=5), back(ld=7), back(ldg=7), back(topk=9), back(offsets=None), back(seqs=0), back(experts=4097, ld=5000, ldg=5000), back(n=-1)]
    assert bad == [capi.ERR_SHAPE] * len(bad)
    assert [back(**{k: 18}) for k in ("logits", "offsets", "counts", "tokens", "grad")] == [capi.ERR_ALIGN] * 5
    null = [back(**{k: None}) for k in ("logits", "counts", "tokens", "grad")]
    assert null == [capi.ERR_NULL] * len(null)


@pytest.mark.parametrize("n", (1, 8, 9, 2368, 2369, 40000))
def test_chunk_numbers_of_sequences_never_meet(n):
    """the rule by which a block finds its chunk: numbers offsets[s] / chunk + s + j, below n / chunk + sequences"""
    import random
    rng = random.Random(n)
    chunk = 8 * min(16, max(1, -(-n // (148 * 2 * 8))))
    for seqs in (1, 2, 5, 64):
        cuts = sorted(rng.choices(range(n + 1), k=seqs - 1))
        off = [0, *cuts, n]
        taken = [off[s] // chunk + s + j for s in range(seqs) for j in range(-(-(off[s + 1] - off[s]) // chunk))]
        assert len(set(taken)) == len(taken) and max(taken) < n // chunk + seqs


@pytest.mark.parametrize("bits", (8, 11))
def test_roundings_of_16_bit_rows(bits):
    """every pair of mantissas of bf16 (8 bits) and fp16 (11): the nearest integer to x * inv, inv = 127 / top rounded up, is the nearest to the quotient
    with halves to the even side, except where 127 divides the mantissa of top and inv is rounded"""
    import numpy as np
    lo, hi = 1 << (bits - 1), 1 << bits
    left = 0
    for top in range(lo, hi):
        inv = np.float32(127.0 / top)
        if float(inv) * top < 127.0:                                   # whole numbers of 35 bits: exact
            inv = np.nextafter(inv, np.float32(np.inf))
        if top % 127 == 0 and float(inv) * top != 127.0:
            left += 1
            continue
        for e in range(0, -11, -1):
            x = np.arange(lo, hi) * 2.0 ** e
            x = x[x <= top]
            m = np.floor(127.0 * x / top)
            a, h = 127.0 * x, (m + 0.5) * top
            want = np.where(a > h, m + 1, np.where(a < h, m, m + m % 2))
            assert np.array_equal(np.rint(x * float(inv)), want), (top, e)
    assert left == (0 if bits == 8 else 7)


def test_row_counts_whose_tiles_pass_32_bits():
    most = (1 << 30) - 1
    for n in (most + 1, (1 << 31) - 1):
        assert lib.b2moe_quantize_rows(16, capi.BF16, 16, n, 16, 16, 16, 16, None) == capi.ERR_SHAPE
        assert lib.b2moe_linear_i8(16, 16, 16, C.byref(bank(1, 1, 16)), n, 16, capi.BF16, 1, None, None) == capi.ERR_SHAPE
        assert lib.b2moe_linear_i8(16, 16, 16, C.byref(bank(1, n, 16)), 1, 16, capi.BF16, n, None, None) == capi.ERR_SHAPE
        assert lib.b2moe_dequant_dump(C.byref(bank(1, n, 16)), 16, None) == capi.ERR_SHAPE
    down = bank(4, 16, 16)
    n = 1 << 29                                                        # two assignments a token and a shared row: 3 * 2^29
    size = lib.b2moe_expert_workspace_bytes(I8, most, 16, capi.F32) * 2
    assert lib.b2moe_expert_down(C.byref(down), C.byref(bank(1, 16, 16)), 16, 16, n, 1, n, 16, 16, size, None) == capi.ERR_SHAPE
