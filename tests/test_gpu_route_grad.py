"""GPU: the gradient of the routing weights on the logits against 64-bit arithmetic, autograd of the routing's definition and differences of it.

Bound, u = 2^-24: dl_j = w_j sum_i v_i (g_j - g_i) (1 - p_j): a difference, a step of the sum (topk of them), the division by the scale, the weight's product, exponential (2), sum and quotient:
(topk + 8) u w_j sum_i v_i |g_j - g_i| (1 - p_j)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U, CLAMP = 2.0 ** -24, 6.103515625e-5


def routed(logits, e, k, gating, norm, scale, bias=None):
    from tqllm_b200 import moe
    if gating == 1:
        ids, w, sw = moe.topk_softmax(logits.cuda(), e, k, scale, shared=logits.shape[1] > e)
        return ids.cpu(), w.cpu(), None if sw is None else sw.cpu()
    ids, w = moe.route_sigmoid(logits.cuda(), e, k, bias, norm, scale)
    return ids.cpu(), w.cpu(), None


def formula(logits, ids, w, g, e, gating, norm, scale):
    """gradient and its bound from the weights as they are"""
    n, k = ids.shape
    l, w, g, at = logits.double(), w.double(), g.double(), ids.long().clamp(0, e - 1)
    live = (ids >= 0) & (ids < e)
    p = torch.sigmoid(l.gather(1, at))
    coupled = torch.full((n, 1), norm or gating == 1)
    if gating == 2 and norm:
        coupled = (p * live).sum(-1, keepdim=True) > CLAMP
    v = w / (scale or 1.0)
    diff = g[:, :, None] - g[:, None, :]
    d = torch.where(coupled, (v[:, None, :] * diff).sum(-1), g)
    size = torch.where(coupled, (v[:, None, :].abs() * diff.abs()).sum(-1), g.abs())
    f = w * (1 - p if gating == 2 else 1.0)
    out, room = torch.zeros(n, e, dtype=torch.float64), torch.zeros(n, e, dtype=torch.float64)
    for s in range(k):
        out.scatter_add_(1, at[:, s : s + 1], (d * f * live)[:, s : s + 1])
        room.scatter_add_(1, at[:, s : s + 1], ((k + 8) * U * size * f.abs() * live)[:, s : s + 1])
    return out, room + 2.0 ** -149


def make(n, e, k, seed, shared=False, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, e + shared, generator=g) * scale, torch.randn(n, k, generator=g), g


CASES = [(1, 1, 1), (1, 4, 2), (5, 33, 7), (48, 32, 4), (130, 512, 10), (3, 4096, 8), (9, 60, 32), (6, 100, 33), (3, 300, 100), (1025, 16, 16)]


@pytest.mark.parametrize("n,e,k", CASES)
@pytest.mark.parametrize("gating,norm", ((1, True), (2, True), (2, False)))
@pytest.mark.parametrize("scale", (0.0, 2.5))
def test_formula(n, e, k, gating, norm, scale):
    from tqllm_b200 import moe
    shared = gating == 1
    logits, g, gen = make(n, e, k, n + e + k, shared)
    ids, w, sw = routed(logits, e, k, gating, norm, scale)
    gs = torch.randn(n, generator=gen) if shared else None
    up = lambda t: None if t is None else t.cuda()
    got = moe.route_backward(logits.cuda(), ids.cuda(), w.cuda(), g.cuda(), e, gating, norm, scale, up(sw), up(gs)).cpu()
    want, room = formula(logits, ids, w, g, e, gating, norm, scale)
    assert bool(((got[:, :e].double() - want).abs() <= room).all())
    chosen = torch.zeros(n, e, dtype=torch.bool).scatter_(1, ids.long(), True)
    assert not got[:, :e][~chosen].any()
    if k == 1 and gating == 1:
        assert not got[:, :e].any()
    if shared:
        s = sw.double()
        assert got.shape[1] == e + 1 and bool(((got[:, e].double() - gs.double() * s * (1 - s)).abs() <= 4 * U * (gs.double() * s * (1 - s)).abs() + 2.0 ** -149).all())
    # added to what is there, in rows of a wider matrix; logits are not needed for softmax
    wide = torch.randn(n, e + 9, generator=gen)
    out = wide.cuda()
    moe.route_backward(logits.cuda() if gating == 2 else None, ids.cuda(), w.cuda(), g.cuda(), e, gating, norm, scale, up(sw), up(gs), out=out[:, : e + shared])
    cols = e + shared
    assert torch.equal(out[:, :cols].cpu(), wide[:, :cols] + got) and torch.equal(out[:, cols:].cpu(), wide[:, cols:])


@pytest.mark.parametrize("gating,norm", ((1, True), (2, True), (2, False)))
def test_autograd_and_differences_of_the_routing(gating, norm):
    """against the definition from the logits on: the weights' own roundings come in, (topk + 60) u of each, so 100 u of the terms"""
    from tqllm_b200 import moe
    n, e, k, scale = 7, 24, 5, 1.5
    logits, g, gen = make(n, e, k, 3)
    ids, w, _ = routed(logits, e, k, gating, norm, scale)
    got = moe.route_backward(logits.cuda(), ids.cuda(), w.cuda(), g.cuda(), e, gating, norm, scale).cpu().double()

    def loss(l):
        p = torch.softmax(l, -1) if gating == 1 else torch.sigmoid(l)
        s = p.gather(1, ids.long())
        if norm:
            s = s / s.sum(-1, keepdim=True).clamp(min=CLAMP)
        return (s * scale * g.double()).sum()
    x = logits.double().requires_grad_()
    want, = torch.autograd.grad(loss(x), x)
    _, room = formula(logits, ids, w, g, e, gating, norm, scale)
    room = room * 100 / (k + 8)
    size = (w.double() * g.double().abs()).sum(-1, keepdim=True).expand(n, e) * 100 * U      # the weights' roundings shift the mean of the gradients too
    assert bool(((got - want).abs() <= room + size).all())
    v = torch.randn(n, e, generator=gen, dtype=torch.float64)
    x = x.detach()
    slope = float(loss(x + 1e-5 * v) - loss(x - 1e-5 * v)) / 2e-5
    assert abs(float((got * v).sum()) - slope) <= float(((room + size) * v.abs()).sum()) + 1e-7


def test_sums_below_the_clamp():
    """sigmoids whose sum is below the clamp are not coupled"""
    from tqllm_b200 import moe
    logits = torch.full((3, 8), -20.0)
    logits[1] = -12.0
    logits[2] = -9.0
    logits += 0.1 * torch.arange(8)
    g = torch.randn(3, 4, generator=torch.Generator().manual_seed(0))
    ids, w, _ = routed(logits, 8, 4, 2, True, 0.0)
    got = moe.route_backward(logits.cuda(), ids.cuda(), w.cuda(), g.cuda(), 8, 2, True, 0.0).cpu().double()
    p = torch.sigmoid(logits.double()).gather(1, ids.long()).sum(-1)
    assert [bool(v) for v in p > CLAMP] == [False, False, True]
    want, room = formula(logits, ids, w, g, 8, 2, True, 0.0)
    assert bool(((got - want).abs() <= room).all())


def test_ids_of_no_expert_and_the_same_expert_twice():
    from tqllm_b200 import moe
    n, e, k = 4, 16, 6
    logits, g, gen = make(n, e, k, 9)
    ids = torch.tensor([[3, 3, 5, -1, 16, 0], [7] * 6, [-1] * 6, [1, 2, 1, 2, 1, 15]], dtype=torch.int32)
    w = torch.rand(n, k, generator=gen)
    for gating, norm in ((1, True), (2, True), (2, False)):
        got = moe.route_backward(logits.cuda(), ids.cuda(), w.cuda(), g.cuda(), e, gating, norm, 0.5).cpu()
        want, room = formula(logits, ids, w, g, e, gating, norm, 0.5)
        assert bool(((got.double() - want).abs() <= room).all())


def test_differences_of_nearly_one_weight():
    """a weight next to one: the difference of its gradient to the others' is what counts, not its own size"""
    from tqllm_b200 import moe
    logits = torch.tensor([[20.0, 0.0, -1.0, 3.0]])
    ids, w, _ = routed(logits, 4, 3, 1, True, 0.0)
    g = torch.tensor([[1e4, 1e4 + 0.25, 1e4 - 0.5]])
    got = moe.route_backward(None, ids.cuda(), w.cuda(), g.cuda(), 4).cpu().double()
    want, room = formula(logits, ids, w, g, 4, 1, True, 0.0)
    assert bool(((got - want).abs() <= room).all()) and float(want.abs().max()) < 1e-6


def test_router_tuning_step():
    """routing weights and balance loss, each gradient by its own call, added into one: as autograd of the whole in 64 bits"""
    from tqllm_b200 import moe
    n, e, k, h, coef = 40, 16, 4, 64, 0.01
    logits, _, gen = make(n, e, k, 5)
    l = logits.cuda()
    ids, w, _ = moe.topk_softmax(l, e, k)
    plan = moe.dispatch(ids, e)
    x = torch.randn(n, h, generator=gen)
    rows, slots = moe.dispatch_rows(x.cuda(), ids, plan)
    mats = torch.randn(e, h, h, generator=gen) / 8
    y = torch.empty_like(rows)
    ends = plan.offsets[: e + 1].tolist()
    for i in range(e):
        y[ends[i] : ends[i + 1]] = rows[ends[i] : ends[i + 1]] @ mats[i].cuda()
    out = moe.combine_rows(y, slots, w, n, k)
    d = torch.randn(n, h, generator=gen)
    gy, gw, _ = moe.combine_rows_backward(d.cuda(), y, slots, w, n, k)
    saved = moe.balance_loss(l, ids, e, coef)
    grad = moe.balance_loss_backward(l, saved, k, coef)
    moe.route_backward(l, ids, w, gw, e, out=grad)
    gr = torch.empty_like(rows)
    for i in range(e):
        gr[ends[i] : ends[i + 1]] = gy[ends[i] : ends[i + 1]] @ mats[i].cuda().t()
    gx = moe.dispatch_rows_backward(gr, slots, n, k)

    lx, xx, sel = logits.double().requires_grad_(), x.double().requires_grad_(), ids.cpu().long()
    p = torch.softmax(lx, -1)
    s = p.gather(1, sel)
    each = torch.stack([xx @ mats[i].double() for i in range(e)], 1)
    want = ((s / s.sum(-1, keepdim=True))[..., None] * each.gather(1, sel[..., None].expand(n, k, h))).sum(1)
    counts = torch.bincount(sel.flatten(), minlength=e).double()
    total = (want * d.double()).sum() + coef * e / (k * n) * (counts * p.mean(0)).sum()
    gl, gxx = torch.autograd.grad(total, (lx, xx))
    # sums of 64 products in 32 bits, of sizes around 8: 1e-4 is 200 u of the largest terms of a sum of this length
    want = want.detach()
    assert float((out.cpu().double() - want).abs().max()) < 1e-4 and float((grad.cpu().double() - gl).abs().max()) < 1e-4 and float((gx.cpu().double() - gxx).abs().max()) < 1e-4
