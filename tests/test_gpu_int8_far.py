"""GPU: 8-bit rows, banks, outputs and logits whose offsets pass 32 bits, looked at near their ends. Bounds as in test_gpu_int8.py and test_gpu_balance.py.
Scales are divided in 64 bits and rounded once: a division by a number in 32 bits is a product with its reciprocal on the device, and off by a unit at times (a quotient of
24 bits by 127 is never within 2^-32 of the middle between two floats, so the two roundings are one)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("60 GB of free device memory are wanted")
    yield
    torch.cuda.empty_cache()


def test_rows_and_outputs():
    from tqllm_b200 import moe
    n, k, m = 70001, 65536, 33000                                      # n k = 4.6e9 values, n m = 2.3e9 outputs
    x = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    far = torch.tensor([0, 32767, 65537, n - 2, n - 1], device="cuda")
    x[far] = torch.randn(5, k, generator=g, device="cuda").bfloat16()
    q, scale = moe.quantize_rows(x)
    rows = x[far].double()
    top = rows.abs().amax(-1, keepdim=True)
    want = torch.round(127.0 * rows / top)
    assert torch.equal(q[far].double(), want) and torch.equal(scale[far].double(), (top / 127.0).float().double()[:, 0]) and int((scale != 0).sum()) == 5
    del x, rows
    w = torch.randint(-127, 128, (m, 32), generator=g, device="cuda", dtype=torch.int8)
    v = torch.rand(m, generator=g, device="cuda")
    y = moe.linear_i8(q[:, :32].contiguous(), torch.ones(n, device="cuda"), moe.DeviceBank.from_int8(w, v), out_dtype=torch.float32)
    exact = (want[:, :32] @ w.double().T) * v.double()
    assert bool(((y[far].double() - exact).abs() <= 2.0 ** -22 * exact.abs()).all()) and not bool(y[1:32767:4001].any())
    far_in = moe.linear_i8(q, torch.ones(n, device="cuda"), moe.DeviceBank.from_int8(torch.ones(3, k, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")), out_dtype=torch.float32)
    assert torch.equal(far_in[far].double(), want.sum(-1, keepdim=True).expand(5, 3))


@pytest.mark.parametrize("n", (2, 100))
def test_banks(n):
    from tqllm_b200 import moe
    e, f, h = 520, 4096, 4096                                          # 8.7e9 weights a bank
    g = torch.Generator("cuda").manual_seed(2)
    used = torch.tensor([0, 127, 128, 256, 511, 519], device="cuda")
    ids = used[torch.rand(n, 6, generator=g, device="cuda").topk(3, -1).indices].int()
    banks = []
    for _ in range(2):
        w = torch.zeros(e, f, h, dtype=torch.int8, device="cuda")
        w[used] = torch.randint(-127, 128, (6, f, h), generator=g, device="cuda", dtype=torch.int8)
        banks.append(moe.DeviceBank.from_int8(w, torch.rand(e, f, generator=g, device="cuda") * 1e-5))
    x = torch.randn(n, h, generator=g, device="cuda")
    plan = moe.dispatch(ids, e)
    act = moe.expert_gateup_swiglu(banks[0], banks[1], x, plan)
    y = moe.expert_down(banks[1], act, plan)
    top = x.double().abs().amax(-1, keepdim=True)
    q, s = torch.round(127.0 * x.double() / top), (top / 127.0).float().double()
    at = act.double().abs().amax(-1, keepdim=True)
    aq, a_s = torch.round(127.0 * act.double() / at), (at / 127.0).float().double()
    for a in list(range(4)) + list(range(3 * n - 2, 3 * n)):
        i, t = int(ids.flatten()[a]), a // 3
        gv, uv = ((b.data[i].double() @ q[t]) * s[t] * b.aux[i].double() for b in banks)
        want = gv / (1 + torch.exp(-gv)) * uv
        assert bool(((act[a].double() - want).abs() <= (4 * gv.abs() + 16) * 2.0 ** -24 * want.abs() + 1e-35).all())
        want = (banks[1].data[i].double() @ aq[a]) * a_s[a] * banks[1].aux[i].double()
        assert bool(((y[a].double() - want).abs() <= 2.0 ** -22 * want.abs() + 1e-35).all())


def test_logits():
    from tqllm_b200 import moe
    n, e = 1050001, 2050                                               # 2.15e9 logits
    g = torch.Generator("cuda").manual_seed(3)
    logits = torch.zeros(n, e, device="cuda")
    logits[-3:] = torch.randn(3, e, generator=g, device="cuda")
    ids = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    ids[-5:] = 7
    b = moe.balance_loss(logits, ids, e, 1.0)
    grad = moe.balance_loss_backward(logits, b, 1, 1.0)
    assert int(b.counts[0, 0]) == n - 5 and int(b.counts[0, 7]) == 5 and int(b.counts.sum()) == n
    p = torch.softmax(logits[-4:].double(), -1)
    c = b.counts[0].double()
    want = p * (c - (p @ c)[:, None]) * e / n ** 2
    size = p * (c + (p @ c)[:, None]) * e / n ** 2
    assert bool(((grad[-4:].double() - want).abs() <= 200 * 2.0 ** -24 * size).all())
    # the mean: n / 128 chunks of 16 rows a warp, an eighth or less of them in turn
    mean = (p[-3:].sum(0) + (n - 3) / e) / n
    assert bool(((b.prob[0].double() - mean).abs() <= (100 + n / 128 / 16) * 2.0 ** -24 * mean).all())
