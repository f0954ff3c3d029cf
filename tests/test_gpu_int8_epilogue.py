"""GPU: 8-bit products with bias, activation and residual in the same pass, against 64-bit arithmetic.

Bound, u = 2^-24: the product has three roundings and the bias one, e = u (3 |product| + |product + bias|). An activation's slope is at most 1.13; its own: SiLU exponential, sum and quotient,
8 u |a|; GELU the complementary error function (8 u) at an argument off by 2 u, which it answers with v^2 times that: (12 + 4 v^2) u |a|; by tanh the exponential of an argument off by
6 u: (8 + 6 |z|) u |a|. The residual's sum: u. Then half a step of the output's type."""
import math

import pytest
import torch

from test_gpu_int8 import linear_case
from test_gpu_int8_waits import DENSE, without_step

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


def activated(name, v):
    if name == "relu":
        return v.clamp(min=0), 0 * v
    if name == "silu":
        a = v * torch.sigmoid(v)
        return a, 8 * a.abs()
    if name == "gelu":
        a = 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
        return a, (12 + 4 * v * v) * a.abs()
    if name == "gelu_tanh":
        z = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
        a = v * torch.sigmoid(z)
        return a, (8 + 6 * z.abs()) * a.abs()
    return v, 0 * v


def check(got, q, s, w, v, bias, name, residual, dtype):
    product = (q.double() @ w.double().t()) * s.double()[:, None] * v.double()
    total = product if bias is None else product + bias.double()
    want, own = activated(name, total)
    room = U * (1.13 * (3 * product.abs() + total.abs()) + own)
    if residual is not None:
        want = want + residual.double()
        room = room + U * (want.abs() + room)
    room = room + HALF[dtype] * (want.abs() + room) + TINY[dtype]
    bad = ~((got.cpu().double() - want).abs() <= room)
    assert not bool(bad.any()), f"{int(bad.sum())}: {got.cpu()[bad][:4]} {want[bad][:4]} {room[bad][:4]}"


def make(n, m, k, seed, dtype):
    q, s, w, v = linear_case(n, m, k, seed)
    s = s / (0.05 * 0.005 * math.sqrt(k) * 73 * 73)                    # products of a size around one
    g = torch.Generator().manual_seed(seed + 1)
    return q, s, w, v, torch.randn(m, generator=g), torch.randn(n, m, generator=g).to(dtype)


# the streaming forms (8 and 16 rows), items of 32 to 128 rows, clusters that share columns, two blocks an SM, pairs
@pytest.mark.parametrize("n,m,k", ((1, 1, 16), (1, 257, 1040), (8, 100, 8192), (3, 4096, 4096), (13, 33, 64), (17, 40, 256), (40, 300, 2560), (77, 1411, 2560), (129, 257, 512), (300, 515, 272), (600, 1411, 2688), (2100, 700, 2048)))
@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("name,bias,residual", (("none", True, False), ("none", False, True), ("relu", True, True), ("silu", False, False), ("gelu", True, True), ("gelu_tanh", False, True)))
def test_epilogue(n, m, k, dtype, name, bias, residual):
    from tqllm_b200 import moe
    q, s, w, v, b, r = make(n, m, k, n + m, dtype)
    bank = moe.DeviceBank.from_int8(w.cuda(), v.cuda())
    b, r = b if bias else None, r if residual else None
    up = lambda t: None if t is None else t.cuda()
    got = moe.linear_i8(q.cuda(), s.cuda(), bank, out_dtype=dtype, bias=up(b), activation=name, residual=up(r))
    check(got, q, s, w, v, b, name, r, dtype)
    if residual:                                                       # the output's own buffer, rows of a wider matrix
        wide = torch.full((n, m + 9), 5.0, dtype=dtype, device="cuda")
        out = wide[:, 4:4 + m]
        out.copy_(r)
        moe.linear_i8(q.cuda(), s.cuda(), bank, out=out, bias=up(b), activation=name, residual=out)
        assert torch.equal(out, got) and bool((wide[:, :4] == 5).all()) and bool((wide[:, 4 + m:] == 5).all())


@pytest.mark.parametrize("family", ("decode", "gemm"))
@pytest.mark.parametrize("n", (5, 40))
def test_forms_agree(family, n):
    """the streaming and the tensor-core form give the bits of the library's own choice"""
    from tqllm_b200 import capi, moe
    q, s, w, v, b, r = make(n, 515, 2560, 3, BF16)
    bank = moe.DeviceBank.from_int8(w.cuda(), v.cuda())
    call = lambda: moe.linear_i8(q.cuda(), s.cuda(), bank, bias=b.cuda(), activation="gelu", residual=r.cuda())
    want = call()
    with capi.family(family):
        assert torch.equal(call(), want)


@pytest.mark.parametrize("name", ("none", "relu", "silu", "gelu", "gelu_tanh"))
@pytest.mark.parametrize("n", (4, 100))
def test_tails_and_what_is_not_finite(name, n):
    """far values of either sign keep their own size; a NaN or an infinity of a scale, a bias or the residual stays in its row, column or place"""
    from tqllm_b200 import moe
    m, k = 64, 256
    q, w = torch.zeros(n, k, dtype=torch.int8), torch.zeros(m, k, dtype=torch.int8)
    q[:, 0], w[:, 0] = 1, 1
    s, v = torch.zeros(n), torch.ones(m)
    bias = torch.linspace(-14, 14, m)
    bank = moe.DeviceBank.from_int8(w.cuda(), v.cuda())
    got = moe.linear_i8(q.cuda(), s.cuda(), bank, out_dtype=F32, bias=bias.cuda(), activation=name)
    check(got, q, s, w, v, bias, name, None, F32)
    for big in (1e5, -1e5, 3e38, -3e38):
        got = moe.linear_i8(q.cuda(), s.cuda(), bank, out_dtype=F32, bias=torch.full((m,), big).cuda(), activation=name)
        assert bool((got == (big if big > 0 or name == "none" else 0.0)).all())
    r = torch.zeros(n, m)
    s[1], bias[7], r[2, 9] = float("nan"), float("nan"), float("inf")
    got = moe.linear_i8(q.cuda(), s.cuda(), bank, out_dtype=F32, bias=bias.cuda(), activation=name, residual=r.cuda()).cpu()
    bad = torch.zeros(n, m, dtype=torch.bool)
    bad[1], bad[:, 7] = True, True
    assert torch.equal(got.isnan(), bad) and got[2, 9].isinf() and bool(got[~bad & (r == 0)].isfinite().all())


@pytest.mark.parametrize("n,m,k,step", DENSE)
def test_unfinished(n, m, k, step):
    """a wait that ran out leaves NaN, also where the residual lies under the output"""
    from tqllm_b200 import moe
    q, s, w, v, b, r = make(n, m, k, 6, BF16)
    bank, out, status = moe.DeviceBank.from_int8(w.cuda(), v.cuda()), r.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    with without_step(step):
        moe.linear_i8(q.cuda(), s.cuda(), bank, out=out, residual=out, bias=b.cuda(), activation="silu", status=status)
    assert bool(torch.isnan(out).all()) and int(status) != 0
    out.copy_(r)
    moe.linear_i8(q.cuda(), s.cuda(), bank, out=out, residual=out, bias=b.cuda(), activation="silu")
    check(out, q, s, w, v, b, "silu", r, BF16)


def test_norm_and_products_in_a_row():
    """the residual stream through two projections, in place, captured and replayed: norm to 8 bits, product with activation, 8 bits again, product with bias onto the stream"""
    from tqllm_b200 import moe
    n, h, f = 24, 512, 1040
    g = torch.Generator().manual_seed(1)
    up, down = (moe.DeviceBank.from_float((torch.randn(a, b, generator=g) / math.sqrt(b)).cuda()) for a, b in ((f, h), (h, f)))
    weight, bias = (1 + 0.1 * torch.randn(h, generator=g)).cuda(), torch.randn(h, generator=g).cuda()
    x, r = torch.randn(n, h, generator=g).to(BF16).cuda(), torch.randn(n, h, generator=g).to(BF16).cuda()
    x0, r0 = x.clone(), r.clone()

    def step():
        norm = moe.rms_norm(x, weight, 1e-6, r, rows=False, quantize=True, sum_out=r)
        mid = moe.linear_i8(norm.q, norm.scale, up, activation="gelu")
        q, s = moe.quantize_rows(mid)
        moe.linear_i8(q, s, down, out=r, bias=bias, residual=r)
        return norm, mid, q, s
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm, mid, q, s = step()
    r.copy_(r0)
    graph.replay()
    torch.cuda.synchronize()
    total = (x0.float() + r0.float()).to(BF16)
    cpu = lambda *t: [v.cpu() for v in t]
    check(mid, *cpu(norm.q, norm.scale, up.data, up.aux), None, "gelu", None, BF16)
    check(r, *cpu(q, s, down.data, down.aux, bias), "none", total.cpu(), BF16)
