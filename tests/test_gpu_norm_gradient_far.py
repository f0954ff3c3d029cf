"""GPU: the norm's gradient of rows at the far ends of 32 bits, through every form: squares that vanish or pass the range, and sums of gradients times rows that pass it.

Bounds. The gradient's as for rows of an ordinary size (the units are powers of two). The weight's gradient: a term is off by 26 u (rho 24, two products); then as many roundings as a term's sum has
steps: the rows of a block (of a warp, and its block's eight warps), the blocks' parts (32 warps of one part at a time, or of four with two steps between the four), five steps between the warps, and
one for what was there before."""
import pytest
import torch

from test_gpu_norm import BF16, F32, U, near

pytestmark = pytest.mark.gpu
EPS = 1e-6


def steps(n, k, dtype, form):
    """roundings of a term's way into the weight's gradient (csrc/norm.cu, launch_norm_grad and norm_weight_grad_k)"""
    up = lambda a, b: -(-a // b)
    V = 4 if dtype is F32 else 8
    by_warp, per_sm = up(k + V - 1 if form == "shifted" else k, 32 * V), max(1, min(8, 16384 // k))
    if form != "single" and by_warp <= 4:
        blocks = min(up(n, 8), 148 * (4 if by_warp <= 2 else 2))
        rows = up(n, 8 * blocks) + 7
    else:
        blocks = min(up(n, 8) * 8, 148 * per_sm // 8 * 8)
        rows = up(n, blocks)
    return rows + (up(blocks, 32) if k % 4 else up(blocks, 128) + 2) + 5 + 1


def definition(h, w, g, s, eps):
    h = h.double()
    a, m = g.double() * w.double(), h.square().mean(-1, keepdim=True) + float(torch.tensor(eps, dtype=F32))
    rho, T = m.rsqrt(), (a * h).abs().mean(-1, keepdim=True) / m
    d = rho * (a - h * (a * h).mean(-1, keepdim=True) / m)
    bound = U * rho * (28 * a.abs() + 119 * h.abs() * T)
    if s is not None:
        d, bound = d + s.double(), bound + 2 * U * s.double().abs()
    return d, bound + 2 * U * d.abs(), g.double() * h * rho


def check(h, w, g, s, eps, got, weight, dtype, form, before=None):
    d, bound, terms = definition(h, w, g, s, eps)
    near(got, d, bound, dtype)
    if weight is None:
        return
    n, k = h.shape
    dw, before = terms.sum(0), 0.0 if before is None else before.double()
    room = (26 + steps(n, k, dtype, form)) * U * terms.abs().sum(0) + U * (dw + before).abs() + 2.0 ** -149
    assert bool(((weight.cpu().double() - dw - before).abs() <= room).all())


def make(n, k, dtype, sizes, seed):
    """rows of these sizes (of h and of the gradient), repeated"""
    gen = torch.Generator().manual_seed(seed)
    h, g, s = torch.randn(n, k, generator=gen), torch.randn(n, k, generator=gen), torch.randn(n, k, generator=gen)
    w = 1 + 0.1 * torch.randn(k, generator=gen)
    for i in range(n):
        a, b = sizes[i % len(sizes)]
        h[i], g[i] = (h[i] * a).clamp(-3e38, 3e38), g[i] * b
    return h.to(dtype), w, g.to(dtype), s.to(dtype)


def place(t, form, other):
    """the same values as rows that begin on 16 bytes, behind them, or (one matrix of the call) elsewhere"""
    if form == "whole":
        return t.cuda()
    begin = 3 if form == "single" and other else 1
    buf = torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")[begin : begin + t.numel()].view(t.shape)
    buf.copy_(t)
    return buf


# a warp a row of one, two and four pieces; a block a row of two pieces a thread and of several; value by value
FORMS = [("whole", n, k) for n, k in ((40, 64), (40, 256), (3000, 128), (40, 512), (1500, 1024), (300, 2048), (30, 4096), (30, 16384))]
FORMS += [("shifted", n, k) for n, k in ((40, 61), (3000, 125), (40, 249), (1500, 501), (300, 2047), (30, 4093), (30, 16381))] + [("single", n, k) for n, k in ((40, 64), (300, 2047), (30, 16381))]
SMALL = ((1.0, 1e-2), (1e-12, 1e-2), (1e-19, 1e-2), (1e-20, 1e-3), (1e-23, 1.0), (1e-30, 1e-2), (3e-38, 1e-8), (1e-39, 1e-8), (1e18, 1.0), (1e30, 1.0))


@pytest.mark.parametrize("form,n,k", FORMS)
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", (0.0, 1e-38, EPS))
@pytest.mark.parametrize("skip", (False, True))
def test_rows_whose_squares_vanish(form, n, k, dtype, eps, skip):
    from tqllm_b200 import moe
    h, w, g, s = make(n, k, dtype, SMALL, n + k)
    s = s if skip else None
    got, weight = moe.rms_norm_backward(place(h, form, False), w.cuda(), place(g, form, False), eps, None if s is None else place(s, form, False), out=place(torch.zeros_like(h), form, True))
    check(h, w, g, s, eps, got, weight, dtype, form)


def test_rows_of_zeros():
    """with eps the gradient is a eps^-1/2, without one it is not a number, in its own row only"""
    from tqllm_b200 import moe
    for form, n, k in FORMS[::3]:
        h, w, g, s = make(n, k, F32, ((1.0, 1.0), (0.0, 1e-3), (1e-25, 1.0)), 5)
        for eps in (EPS, 1e-38):
            got, weight = moe.rms_norm_backward(place(h, form, False), w.cuda(), place(g, form, False), eps, out=place(torch.zeros_like(h), form, True))
            check(h, w, g, None, eps, got, weight, F32, form)
        got, _ = moe.rms_norm_backward(place(h, form, False), w.cuda(), place(g, form, False), 0.0, out=place(torch.zeros_like(h), form, True), weight_grad=False)
        zero = (h == 0).all(-1)
        assert bool(got.cpu()[zero].isnan().all())
        d, bound, _ = definition(h[~zero], w, g[~zero], None, 0.0)
        near(got.cpu()[~zero], d, bound, F32)
