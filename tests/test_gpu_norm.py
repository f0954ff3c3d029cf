"""GPU: the norm of rows, its 8-bit output and its gradient against 64-bit arithmetic, and the gradient against differences of the definition.

Bounds, with u = 2^-24. The norm: a thread sums 32 squares, trees of 10 steps the threads: the mean is off by 44 u with its division and eps, its root by half of that, rho by 24 u with root
and quotient, and y by two products more: 26 u of itself, then half a step of its own type. The scale: 24 u, the largest product, a product and a quotient: 27 u. The integers are exact.
The gradient: a = g w is off by u, c = sum of a h by 45 u sum|a h|, t = c / k / m by 45 u of T = sum|a h| / (k m) and 46 u of itself (|t| <= T), so
d = rho (a - h t) + s by (24 + 4) u rho |a| + (24 + 91 + 4) u rho |h| T + 2 u |s|, then half a step. A term of the weight's gradient is off by 27 u; a block adds its rows one by one, then eight threads
the blocks' parts: rows / blocks + blocks / 8 + 8."""
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}
EPS = 1e-6


def make(n, k, dtype, wdtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, k, generator=g) * scale
    x[:, :: max(1, k // 7)] *= 8
    r = torch.randn(n, k, generator=g) * 2 * scale
    w = 1 + 0.1 * torch.randn(k, generator=g)
    return x.to(dtype), r.to(dtype), w.to(wdtype), g


def root(h):
    return (h.square().mean(-1, keepdim=True) + EPS).sqrt()


def near(got, want, bound, dtype):
    """got (of dtype) within the bound of want, and half a step of its type"""
    got = got.cpu().double()
    room = bound + HALF[dtype] * (want.abs() + bound) + TINY[dtype]
    bad = ~((got - want).abs() <= room)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}: {got[bad][:4]} {want[bad][:4]} {room[bad][:4]}"


def integers(u):
    """the nearest integers to 127 u / max|u| of a row, exactly"""
    top = u.abs().amax(-1, keepdim=True)
    t = 127.0 * u / torch.where(top > 0, top, torch.ones_like(top))
    q = torch.round(t)
    close = ((t - torch.floor(t)) - 0.5).abs() < 1e-6
    for i, j in close.nonzero().tolist():
        f = Fraction(127) * Fraction(float(u[i, j])) / Fraction(float(top[i, 0]))
        q[i, j] = round(f)
    return q


def check_norm(x, r, w, out, dtype):
    h = (x.float() if r is None else x.float() + r.float()).double()
    if out.sum is not None:
        assert torch.equal(out.sum.cpu(), h.float().to(dtype))
    if out.y is not None:
        want = h / root(h) * w.double()
        near(out.y, want, 26 * U * want.abs(), dtype)
    if out.q is not None:
        v = h * w.double()
        assert torch.equal(out.q.cpu().double(), integers(v))
        want = (v.abs().amax(-1, keepdim=True) / root(h) / 127)[:, 0]
        assert bool(((out.scale.cpu().double() - want).abs() <= 27 * U * want + 2.0 ** -149).all())


def up(t):
    return None if t is None else t.cuda()


# a row of one value, odd ones, a piece a lane, around the limits of the forms (a warp a row, pieces a thread, 512 threads), many rows
@pytest.mark.parametrize("n,k", ((1, 1), (3, 7), (2, 33), (5, 127), (1, 2049), (3, 8193), (2, 16383), (2500, 101), (1, 16), (4, 64), (7, 1024), (3, 1040), (2, 4096), (1, 4112), (3, 8192), (2, 8208), (2, 16384),
                                 (2368, 128), (2400, 1024), (2500, 2064), (2369, 512)))
@pytest.mark.parametrize("dtype,wdtype", ((BF16, F32), (BF16, BF16), (F16, F32), (F16, F16), (F32, F32)))
@pytest.mark.parametrize("residual", (False, True))
def test_norm(n, k, dtype, wdtype, residual):
    from tqllm_b200 import moe
    x, r, w, _ = make(n, k, dtype, wdtype, 7 * n + k)
    r = r if residual else None
    check_norm(x, r, w, moe.rms_norm(x.cuda(), w.cuda(), EPS, up(r)), dtype)
    if k % 16 == 0:
        both = moe.rms_norm(x.cuda(), w.cuda(), EPS, up(r), quantize=True)
        check_norm(x, r, w, both, dtype)
        only = moe.rms_norm(x.cuda(), w.cuda(), EPS, up(r), rows=False, quantize=True)
        assert only.y is None and torch.equal(only.q, both.q) and torch.equal(only.scale, both.scale)


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
def test_halves(dtype):
    """rows whose quotients are halves: 127 u / top = m + 1/2, where 127 divides (2 m + 1) u; and products that round to the same 32 bits, of which the larger one counts"""
    from tqllm_b200 import moe
    x = torch.zeros(4, 128, dtype=dtype)
    x[0] = torch.arange(128) / 2.0 - 32
    x[0, 0], x[0, 1], x[0, 2] = 127.0, 63.5, -63.5
    x[1, :4] = torch.tensor([2.0, 1.0, -1.0, 0.5])
    x[2] = 1.0
    x[3, 5] = -3.0
    w = torch.ones(128)
    check_norm(x, None, w, moe.rms_norm(x.cuda(), w.cuda(), EPS, quantize=True), dtype)
    g = torch.Generator().manual_seed(1)
    w = torch.randint(1, 128, (128,), generator=g).float()
    x = torch.randint(-64, 65, (64, 128), generator=g).to(dtype)
    check_norm(x, None, w, moe.rms_norm(x.cuda(), w.cuda(), EPS, quantize=True), dtype)
    # h w just around its largest: one step of 32 bits apart before rounding
    w = torch.nextafter(torch.full((128,), 1.3), torch.tensor(2.0)) + 2.0 ** -23 * torch.arange(128)
    x = torch.full((8, 128), 1.7).to(dtype)
    x[:, 64:] *= torch.tensor(0.5)
    check_norm(x, None, w, moe.rms_norm(x.cuda(), w.cuda(), EPS, quantize=True), dtype)


def test_rows_at_the_edges_of_the_types():
    """zeros, infinities and NaN, squares and products that pass 32 bits, products below their range"""
    from tqllm_b200 import moe
    x = torch.zeros(9, 256)
    g = torch.Generator().manual_seed(3)
    x[1] = torch.randn(256, generator=g)
    x[1, 9] = float("inf")
    x[2] = torch.randn(256, generator=g)
    x[2, 200] = float("nan")
    x[3] = torch.randn(256, generator=g) * 2e37
    x[4] = 3.3e38
    x[5] = torch.randn(256, generator=g) * 1e-30
    x[6] = torch.randn(256, generator=g) * 1e-38
    x[7] = torch.randn(256, generator=g)
    x[8, 17] = 1e-44
    w = 1 + 0.1 * torch.randn(256, generator=g)
    out = moe.rms_norm(x.cuda(), w.cuda(), EPS, quantize=True)
    y, q, scale = out.y.cpu(), out.q.cpu(), out.scale.cpu()
    assert not y[0].any() and not q[0].any() and scale[0] == 0
    assert y[1, 9].isnan() and not y[1, :9].any() and scale[1].isnan() and not q[1].any()
    assert y[2].isnan().all() and scale[2].isnan() and not q[2].any()
    h = x.double()
    want = h / root(h) * w.double()
    keep = [0, 3, 4, 5, 6, 7, 8]
    near(y[keep], want[keep], 28 * U * want[keep].abs() + 2.0 ** -149, F32)
    fine = [3, 5, 7]
    v = (h * w.double())[fine]
    assert torch.equal(q[fine].double(), integers(v))
    assert bool(((h * w.double())[4] > 3.41e38).any()) and scale[4].isnan() and not q[4].any()
    top = v.abs().amax(-1) / root(h)[fine, 0] / 127
    assert bool(((scale[fine].double() - top).abs() <= 29 * U * top).all())
    for h, w in ((1e30, 1e10), (1e10, 1e30)):                              # products beyond 32 bits, with and without the squares
        out = moe.rms_norm(torch.full((1, 256), h).cuda(), torch.full((256,), w).cuda(), EPS, quantize=True)
        assert not out.q.any() and out.scale.isnan().all() and bool(((out.y / w - 1).abs() < 1e-6).all())


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("k", (64, 65))
def test_rows_of_wider_matrices(dtype, k):
    """strides, outputs that are given, what lies beside the rows stays, outputs on inputs"""
    from tqllm_b200 import moe
    n = 6
    x, r, w, _ = make(n, k, dtype, F32, 5)
    wide = [torch.full((n, 96), 7.0, dtype=dtype, device="cuda") for _ in range(4)]
    wide[0][:, 8:8 + k], wide[1][:, 16:16 + k] = x.cuda(), r.cuda()
    y, s = wide[2][:, 24:24 + k], wide[3][:, :k]
    out = moe.rms_norm(wide[0][:, 8:8 + k], w.cuda(), EPS, wide[1][:, 16:16 + k], out=y, sum_out=s)
    assert out.y.data_ptr() == y.data_ptr() and out.sum.data_ptr() == s.data_ptr()
    check_norm(x, r, w, out, dtype)
    assert bool((wide[2][:, :24] == 7).all()) and bool((wide[2][:, 24 + k:] == 7).all()) and bool((wide[3][:, k:] == 7).all())
    a, b = x.cuda(), r.cuda()
    out = moe.rms_norm(a, w.cuda(), EPS, b, out=a, sum_out=b)
    check_norm(x, r, w, out, dtype)


def gradient(h, w, g, s):
    h = h.double()
    a, m = g.double() * w.double(), h.square().mean(-1, keepdim=True) + EPS
    rho, T = m.rsqrt(), (a * h).abs().mean(-1, keepdim=True) / m
    d = rho * (a - h * (a * h).mean(-1, keepdim=True) / m)
    bound = U * rho * (28 * a.abs() + 119 * h.abs() * T)
    if s is not None:
        d, bound = d + s.double(), bound + 2 * U * s.double().abs()
    terms = g.double() * h * rho
    return d, bound + 2 * U * d.abs(), terms.sum(0), terms.abs().sum(0)


def check_gradient(h, w, g, s, got, weight, dtype, before=None):
    d, bound, dw, size = gradient(h, w, g, s)
    near(got, d, bound, dtype)
    n, k = h.shape
    blocks = min((n + 7) // 8 * 8, 148 * max(1, min(8, 8192 // k)) // 8 * 8)
    before = 0.0 if before is None else before.double()
    room = (27 + n // blocks + 1 + blocks // 8 + 10) * U * size + U * (dw + before).abs() + 2.0 ** -149
    assert bool(((weight.cpu().double() - dw - before).abs() <= room).all())


@pytest.mark.parametrize("n,k", ((1, 1), (3, 7), (5, 127), (1, 2049), (3, 8193), (2, 16383), (2500, 101), (1, 16), (4, 64), (7, 1024), (300, 1040), (2, 2048), (160, 4096), (3, 8192), (2, 8208), (150, 16384), (2400, 512)))
@pytest.mark.parametrize("dtype,wdtype", ((BF16, F32), (BF16, BF16), (F16, F32), (F16, F16), (F32, F32)))
@pytest.mark.parametrize("skip", (False, True))
def test_gradient(n, k, dtype, wdtype, skip):
    from tqllm_b200 import moe
    x, r, w, gen = make(n, k, dtype, wdtype, 3 * n + k)
    g = torch.randn(n, k, generator=gen).to(dtype)
    s = r if skip else None
    got, weight = moe.rms_norm_backward(x.cuda(), w.cuda(), g.cuda(), EPS, up(s))
    check_gradient(x, w, g, s, got, weight, dtype)
    again, none = moe.rms_norm_backward(x.cuda(), w.cuda(), g.cuda(), EPS, up(s), weight_grad=False)
    assert none is None and torch.equal(again, got)


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("k,ld,begin", ((1, 1, 0), (1, 1, 3), (2, 3, 1), (5, 5, 7), (33, 48, 3), (101, 101, 5), (101, 108, 5), (1031, 1040, 1), (2050, 2051, 7), (5000, 5002, 2), (8193, 8193, 1), (16370, 16371, 6), (64, 72, 4), (64, 64, 1), (4096, 4099, 0)))
def test_rows_that_begin_anywhere(dtype, k, ld, begin):
    """rows that begin behind 16 bytes, in all matrices alike or in one otherwise; nothing beside them is touched"""
    from tqllm_b200 import moe
    n = 19
    x, r, w, gen = make(n, k, dtype, F32, k + ld)
    g = torch.randn(n, k, generator=gen).to(dtype)
    for lone in (None, 0, 4):
        bufs = [torch.full((n * ld + 16,), 3.0, dtype=dtype, device="cuda") for _ in range(8)]
        view = [b[begin + (i == lone):].as_strided((n, k), (ld, 1)) for i, b in enumerate(bufs)]
        for v, t in zip(view, (x, r, x, r, x, g, r, x)):
            v.copy_(t)
        keep = [b.clone() for b in bufs]
        out = moe.rms_norm(view[0], w.cuda(), EPS, view[1], out=view[2], sum_out=view[3])
        check_norm(x, r, w, out, dtype)
        check_norm(x, None, w, moe.rms_norm(view[0], w.cuda(), EPS, out=view[2]), dtype)
        got, weight = moe.rms_norm_backward(view[4], w.cuda(), view[5], EPS, view[6], out=view[7])
        got = got.clone()
        check_gradient(x, w, g, r, got, weight, dtype)
        for i, (b, v, t) in enumerate(zip(bufs, view, (x, r, x, r, x, g, r, x))):
            v.copy_(t)
            assert torch.equal(b, keep[i])
        moe.rms_norm_backward(view[4], w.cuda(), view[5], EPS, view[6], out=view[5])
        assert torch.equal(view[5], got) if lone is None else True


def test_gradient_is_added_and_lies_on_its_inputs():
    from tqllm_b200 import moe
    x, r, w, gen = make(33, 640, BF16, F32, 11)
    g = torch.randn(33, 640, generator=gen).to(BF16)
    for place in range(3):
        a, b, c = x.cuda(), g.cuda(), r.cuda()
        before = torch.randn(640, generator=gen)
        weight = before.cuda()
        got, same = moe.rms_norm_backward(a, w.cuda(), b, EPS, c, out=(a, b, c)[place], grad_weight=weight)
        assert got.data_ptr() == (a, b, c)[place].data_ptr() and same is weight
        check_gradient(x, w, g, r, got, weight, BF16, before)
        two = moe.rms_norm_backward(x.cuda(), w.cuda(), g.cuda(), EPS, r.cuda())
        three = moe.rms_norm_backward(x.cuda(), w.cuda(), g.cuda(), EPS, r.cuda())
        assert all(torch.equal(p, q) for p, q in zip(two, three))


def test_gradient_of_rows_beyond_32_bit_squares():
    from tqllm_b200 import moe
    x, _, w, gen = make(4, 256, F32, F32, 2)
    x[1] *= 1e30
    x[2] = 0
    g = torch.randn(4, 256, generator=gen)
    got, weight = moe.rms_norm_backward(x.cuda(), w.cuda(), g.cuda(), EPS)
    check_gradient(x, w, g, None, got, weight, F32)


def test_gradient_against_differences():
    """central differences of the definition in 64 bits, step 1e-4: off by the third derivative times 1e-8 / 6 and 1e-12 of rounding, 1e-6 in all for rows of this size"""
    from tqllm_b200 import moe
    x, _, w, gen = make(3, 48, F32, F32, 4, 0.5)
    g, v, vw = torch.randn(3, 48, generator=gen), torch.randn(3, 48, generator=gen).double(), torch.randn(48, generator=gen).double()
    got, weight = moe.rms_norm_backward(x.cuda(), w.cuda(), g.cuda(), EPS)
    f = lambda h, w: float((h / root(h) * w * g.double()).sum())
    h, ww, e = x.double(), w.double(), 1e-4
    slope = (f(h + e * v, ww) - f(h - e * v, ww)) / (2 * e)
    _, bound, dw, size = gradient(x, w, g, None)
    assert abs(float((got.cpu().double() * v).sum()) - slope) <= float(((bound + U * got.cpu().double().abs()) * v.abs()).sum()) + 1e-6
    slope = (f(h, ww + e * vw) - f(h, ww - e * vw)) / (2 * e)
    assert abs(float((weight.cpu().double() * vw).sum()) - slope) <= float((40 * U * size * vw.abs()).sum()) + 1e-6


def test_offsets_beyond_32_bits():
    """rows of a matrix of more than 2^32 values: the last one is found"""
    from tqllm_b200 import moe
    n, k, ld = 3, 64, (1 << 31) + 64
    buf = torch.zeros(2 * ld + k, dtype=BF16, device="cuda")
    x = buf.as_strided((n, k), (ld, 1))
    a, _, w, _ = make(n, k, BF16, F32, 8)
    x.copy_(a)
    check_norm(a, None, w, moe.rms_norm(x, w.cuda(), EPS, quantize=True), BF16)
    g = torch.randn(n, k).to(BF16)
    got, weight = moe.rms_norm_backward(x, w.cuda(), g.cuda(), EPS)
    check_gradient(a, w, g, None, got, weight, BF16)


def test_captured():
    """a captured step replays with new inputs; two graphs and an eager call in between share nothing"""
    from tqllm_b200 import moe
    x, r, w, gen = make(9, 512, BF16, F32, 21)
    xs, rs, ws = x.cuda(), r.cuda(), w.cuda()
    gs = torch.randn(9, 512, generator=gen).to(BF16).cuda()

    def step():
        out = moe.rms_norm(xs, ws, EPS, rs, quantize=True)
        return out, moe.rms_norm_backward(out.sum, ws, gs, EPS, gs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
        graphs.append((graph, got))
    for seed in (1, 2):
        a, b, _, _ = make(9, 512, BF16, F32, seed)
        xs.copy_(a)
        rs.copy_(b)
        for graph, _ in graphs:
            graph.replay()
        step()
        torch.cuda.synchronize()
        for _, (out, (grad, weight)) in graphs:
            check_norm(a, b, w, out, BF16)
            check_gradient(out.sum.cpu(), w, gs.cpu(), gs.cpu(), grad, weight, BF16)


def test_zero_rows_without_eps():
    """0 / sqrt(0) is not a number; the 8-bit row of zeros has scale 0 all the same"""
    from tqllm_b200 import moe
    x = torch.zeros(2, 64)
    x[1] = 1.0
    out = moe.rms_norm(x.cuda(), torch.ones(64).cuda(), 0.0, quantize=True)
    assert out.y[0].isnan().all() and not out.q[0].any() and out.scale[0] == 0
    assert bool((out.y[1] == 1).all()) and bool((out.q[1] == 127).all())


def test_long_batches():
    """more rows than a launch has blocks, in every form of the gradient"""
    from tqllm_b200 import moe
    for n, k, dtype in ((30011, 64, BF16), (20000, 77, F16), (9001, 520, F32), (3001, 2056, BF16), (2003, 4099, F32)):
        x, r, w, gen = make(n, k, dtype, F32, n)
        g = torch.randn(n, k, generator=gen).to(dtype)
        got, weight = moe.rms_norm_backward(x.cuda(), w.cuda(), g.cuda(), EPS, r.cuda())
        check_gradient(x, w, g, r, got, weight, dtype)
        check_norm(x, r, w, moe.rms_norm(x.cuda(), w.cuda(), EPS, r.cuda()), dtype)
