"""GPU: rows of tokens sorted by expert, rows of slots back with their weights, and the gradients of both, against 64-bit arithmetic. Rows and slots have to be equal.

Bounds, u = 2^-24: a sum of m terms in 32 bits is off by m u of the terms' sizes (one rounding a product and sum), then half a step of the type. A product of rows: a thread adds at most
hidden / 256 + 8 terms (hidden / 32 of short rows), trees and warps 13: hidden / 32 + 32. A row's gradient: one product."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


def near(got, want, bound, dtype):
    got = got.cpu().double()
    room = bound + HALF[dtype] * (want.abs() + bound) + TINY[dtype]
    bad = ~((got - want).abs() <= room)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}: {got[bad][:4]} {want[bad][:4]} {room[bad][:4]}"


def make(n, h, e, k, dtype, seed, skip=0.0, one=False):
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(n, e, generator=g).topk(k, -1).indices.int()
    if one:
        ids[:, 0] = e // 2                                             # an expert with a row of every token
        ids[:, 1:] = torch.where(ids[:, 1:] == e // 2, -1, ids[:, 1:])
    ids[torch.rand(n, k, generator=g) < skip] = -1
    x = torch.randn(n, h, generator=g).to(dtype)
    w = torch.rand(n, k, generator=g) + 0.1
    return ids, x, w, torch.rand(n, generator=g), g


def sorted_plain(ids, e, shared):
    """slot of every assignment (those of the shared expert last), and the token of every slot"""
    n, k = ids.shape
    flat = ids.flatten().tolist()
    order = sorted((a for a in range(n * k) if 0 <= flat[a] < e), key=lambda a: (flat[a], a)) + [n * k + t for t in range(n) if shared]
    slots = torch.full((n * k + (n if shared else 0),), -1, dtype=torch.int32)
    for s, a in enumerate(order):
        slots[a] = s
    return slots, torch.tensor([a // k if a < n * k else a - n * k for a in order], dtype=torch.long)


CASES = [dict(n=1, h=8, e=1, k=1), dict(n=1, h=2048, e=512, k=10), dict(n=3, h=40, e=5, k=2), dict(n=64, h=2048, e=64, k=10), dict(n=33, h=264, e=7, k=7, skip=0.5), dict(n=129, h=1032, e=3, k=1),
         dict(n=40, h=16, e=8, k=2, skip=1.0), dict(n=700, h=72, e=9, k=3, one=True), dict(n=2500, h=24, e=4, k=2, one=True), dict(n=20, h=136, e=60, k=40), dict(n=5, h=4104, e=16, k=4), dict(n=2, h=16392, e=40, k=33),
         dict(n=1300, h=40, e=60, k=40, skip=0.3), dict(n=1190, h=1096, e=50, k=35, skip=0.1), dict(n=1500, h=520, e=70, k=9), dict(n=1184, h=8, e=2, k=1, skip=1.0)]


def run(case, dtype, shared, weights=True):
    from tqllm_b200 import moe
    n, e, k = case["n"], case["e"], case["k"]
    ids, x, w, sw, g = make(dtype=dtype, seed=case["n"] + case["h"], **{"skip": 0.0, **case})
    plan = moe.dispatch(ids.cuda(), e, n if shared else 0)
    rows = torch.full((n * k + (n if shared else 0), case["h"]), 9.0, dtype=dtype, device="cuda")
    rows, slots = moe.dispatch_rows(x.cuda(), ids.cuda(), plan, rows=rows)
    return moe, ids, x, w, sw if shared else None, g, rows, slots


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("shared", (False, True))
def test_there_and_back(case, dtype, shared):
    moe, ids, x, w, sw, g, rows, slots = run(case, dtype, shared)
    want, token = sorted_plain(ids, case["e"], shared)
    assert torch.equal(slots.cpu(), want)
    live = token.numel()
    assert torch.equal(rows[:live].cpu(), x[token]) and bool((rows[live:] == 9).all())
    n, k, h = case["n"], case["k"], case["h"]
    y = torch.randn(rows.shape, generator=g).to(dtype)
    y[live:] = float("nan")                                            # rows of no assignment are not looked at
    r = torch.randn(n, h, generator=g).to(dtype)
    for weights, shared_weights, residual in ((w, sw, r), (w, None, None), (None, None, r)):
        up = lambda t: None if t is None else t.cuda()
        got = moe.combine_rows(y.cuda(), slots, up(weights), n, k, shared_weights=up(shared_weights), residual=up(residual))
        total, size = plain_back(y, want, weights, shared_weights, residual, n, k, shared)
        near(got, total, (k + 3) * U * size, dtype)
    got = moe.dispatch_rows_backward(y.cuda(), slots, n, k)
    total, size = plain_back(y, want, None, None, None, n, k, shared)
    near(got, total, (k + 3) * U * size, dtype)


def plain_back(y, slots, w, sw, r, n, k, shared):
    h = y.shape[1]
    total = torch.zeros(n, h, dtype=torch.float64) if r is None else r.double()
    size = total.abs()
    for s in range(k + (1 if shared else 0)):
        at = (slots[: n * k].view(n, k)[:, s] if s < k else slots[n * k :]).long()
        t = (at >= 0).nonzero()[:, 0]
        f = torch.ones(n) if (w if s < k else sw) is None else w[:, s] if s < k else sw
        term = f.double()[t, None] * y.double()[at[t]]
        total[t] += term
        size[t] += term.abs()
    return total, size


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("shared", (False, True))
def test_gradients(case, dtype, shared):
    moe, ids, x, w, sw, g, rows, slots = run(case, dtype, shared)
    n, k, h = case["n"], case["k"], case["h"]
    want, token = sorted_plain(ids, case["e"], shared)
    live = token.numel()
    y = torch.randn(rows.shape, generator=g).to(dtype)
    y[live:] = float("inf")
    d = torch.randn(n, h, generator=g).to(dtype)
    up = lambda t: None if t is None else t.cuda()
    grad_y = torch.full_like(rows, 5.0)
    gy, gw, gs = moe.combine_rows_backward(d.cuda(), y.cuda(), slots, w.cuda(), n, k, shared_weights=up(sw), grad_y=grad_y)
    assert gy is grad_y and bool((gy[live:] == 5).all()) and (gs is not None) == shared
    weight = torch.cat([w.flatten()] + ([sw] if shared else [])).double()
    of = torch.full((rows.shape[0],), -1, dtype=torch.long)             # assignment of the slot
    of[want[want >= 0].long()] = (want >= 0).nonzero()[:, 0]
    if live:
        near(gy[:live], weight[of[:live], None] * d.double()[token], U * (weight[of[:live], None] * d.double()[token]).abs(), dtype)
    terms = d.double()[token] * y.double()[:live]
    dots, size = torch.zeros(weight.numel(), dtype=torch.float64), torch.zeros(weight.numel(), dtype=torch.float64)
    dots[of[:live]], size[of[:live]] = terms.sum(-1), terms.abs().sum(-1)
    got = torch.cat([gw.cpu().flatten()] + ([gs.cpu()] if shared else [])).double()
    assert bool(((got - dots).abs() <= (h / 32 + 32) * U * size).all())
    # the rows themselves as the gradient's buffer, weights of one
    z = y.cuda()
    z, gw2, _ = moe.combine_rows_backward(d.cuda(), z, slots, None, n, k, grad_y=z)
    assert torch.equal(gw2, gw) and torch.equal(z[:live].cpu(), d[token]) and bool(z[live:].isinf().all())


def test_against_differences():
    """the loss sum(out * c) of the way there and back is linear in every input: central differences of the 64-bit definition, step 1/2, give its gradients but for the roundings"""
    case = dict(n=6, h=40, e=5, k=3, skip=0.2)
    moe, ids, x, w, sw, g, rows, slots = run(case, F32, True)
    n, k, h = 6, 3, 40
    want, token = sorted_plain(ids, 5, True)
    y, c = torch.randn(rows.shape, generator=g), torch.randn(n, h, generator=g)
    gy, gw, gs = moe.combine_rows_backward(c.cuda(), y.cuda(), slots, w.cuda(), n, k, shared_weights=sw.cuda())
    f = lambda y, w, sw: float((plain_back(y, want, w, sw, None, n, k, True)[0] * c.double()).sum())
    y, w, sw = y.double(), w.double(), sw.double()
    for i in range(8):
        v = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (y, w, sw)]
        slope = f(y + v[0] / 2, w, sw) - f(y - v[0] / 2, w, sw)
        got = float((gy.cpu().double() * v[0]).sum())
        assert abs(got - slope) <= 2 * U * float((gy.cpu().double() * v[0]).abs().sum()) + 1e-9
        slope = f(y, w + v[1] / 2, sw) - f(y, w - v[1] / 2, sw)
        room = 40 * U * float(sum((c.double()[t].abs() * y[s].abs()).sum() * v[1].abs().max() for s, t in enumerate(token)))
        assert abs(float((gw.cpu().double() * v[1]).sum()) - slope) <= room
        slope = f(y, w, sw + v[2] / 2) - f(y, w, sw - v[2] / 2)
        assert abs(float((gs.cpu().double() * v[2]).sum()) - slope) <= room / float(v[1].abs().max()) * float(v[2].abs().max())


def test_plans_in_another_order_and_repeated_experts():
    """a plan from groups, whose lists are in any order: the slots are the plan's; and a token that names an expert twice has two rows there"""
    from tqllm_b200 import moe
    from tqllm_b200.capi import check, lib
    n, k, e, h = 100, 2, 3, 64
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(-1, e, (n, k), generator=g, dtype=torch.int32)
    ids[7] = 1
    x = torch.randn(n, h, generator=g).to(BF16)
    plan = moe.dispatch(ids.cuda(), e)
    rows, slots = moe.dispatch_rows(x.cuda(), ids.cuda(), plan)
    want, token = sorted_plain(ids, e, False)
    assert torch.equal(slots.cpu(), want) and torch.equal(rows[: token.numel()].cpu(), x[token])
    assert not rows[token.numel():].any()
    counts = torch.zeros(e, dtype=torch.int32)
    groups = torch.full((e, n * k), -1, dtype=torch.int32)
    for a in torch.randperm(n * k, generator=g).tolist():
        i = int(ids.flatten()[a])
        if i >= 0:
            groups[i, counts[i]] = a
            counts[i] += 1
    other = moe.Plan(e, n, k, 0, "cuda")
    on = counts.cuda(), groups.cuda()
    check(lib.b2moe_plan_from_groups(on[0].data_ptr(), on[1].data_ptr(), n * k, e, n * k, other.buf.data_ptr(), torch.cuda.current_stream().cuda_stream), "groups")
    rows, slots = moe.dispatch_rows(x.cuda(), ids.cuda(), other)
    perm = torch.cat([groups[i, : counts[i]] for i in range(e)]).long()
    want = torch.full((n * k,), -1, dtype=torch.int32)
    want[perm] = torch.arange(perm.numel(), dtype=torch.int32)
    assert torch.equal(slots.cpu(), want) and torch.equal(rows[: perm.numel()].cpu(), x[perm // k])


@pytest.mark.parametrize("n", (30, 1300))
def test_shared_expert_for_a_part_of_the_tokens(n):
    """the plan of a rank that evaluates the shared expert for its own tokens: the others have no shared slot"""
    from tqllm_b200 import capi, moe
    from tqllm_b200.capi import check, lib
    k, e, h, first, count = 3, 7, 64, 5, 11
    ids, x, w, sw, g = make(n, h, e, k, BF16, 3, skip=0.4)
    di, dx = ids.cuda(), x.cuda()
    plan = moe.Plan(e, n, k, count, "cuda")
    ws = torch.empty(max(16, lib.b2moe_dispatch_workspace_bytes(e, n * k)), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    check(lib.b2moe_dispatch_range(di.data_ptr(), n, k, e, first, count, plan.buf.data_ptr(), ws.data_ptr(), ws.numel(), stream), "range")
    rows, slots = moe.dispatch_rows(dx, di, plan)
    routed, token = sorted_plain(ids, e, False)
    live = token.numel()
    want = torch.cat([routed, torch.full((n,), -1, dtype=torch.int32)])
    want[n * k + first : n * k + first + count] = torch.arange(live, live + count, dtype=torch.int32)
    assert slots.numel() == n * k + n and torch.equal(slots.cpu(), want)
    assert torch.equal(rows[:live].cpu(), x[token]) and torch.equal(rows[live : live + count].cpu(), x[first : first + count]) and not rows[live + count :].any()
    out = moe.combine_rows(rows, slots, w.cuda(), n, k, shared_weights=sw.cuda())
    total, size = plain_back(rows.cpu(), want, w, sw, None, n, k, True)
    near(out, total, (k + 3) * U * size, BF16)
    gy, gw, gs = moe.combine_rows_backward(dx, rows, slots, w.cuda(), n, k, shared_weights=sw.cuda())
    own = torch.zeros(n, dtype=torch.bool)
    own[first : first + count] = True
    assert not gs.cpu()[~own].any() and bool((gs.cpu()[own] > 0).all())


def test_slots_that_lead_nowhere_and_ids_of_another_plan():
    """slots outside the rows are left out; ids that the plan was not made of find no slot, or that of the plan"""
    from tqllm_b200 import moe
    n, k, e, h = 9, 2, 4, 32
    ids, x, w, _, g = make(n, h, e, k, F32, 1)
    plan = moe.dispatch(ids.cuda(), e)
    _, slots = moe.dispatch_rows(x.cuda(), (ids + 1).cuda(), plan)
    assert bool((slots == -1).all())
    y = torch.randn(n * k, h, generator=g).cuda()
    bad = torch.tensor([n * k, -7, 1 << 30, -(1 << 31), 3, n * k + 5], dtype=torch.int32).repeat(3).cuda()
    out = moe.combine_rows(y, bad, w.cuda(), n, k)
    gy, gw, _ = moe.combine_rows_backward(x.cuda(), y, bad, w.cuda(), n, k)
    want = torch.zeros(n, h)
    for t in (2, 5, 8):
        want[t] = y[3].cpu() * w[t, 0]
    assert torch.equal(out.cpu(), want)
    assert bool((gw.cpu()[[0, 1, 3, 4, 6, 7]] == 0).all()) and not gy[torch.arange(n * k) != 3].any()


def test_wider_matrices():
    """strided rows; what lies beside them stays; residual in place"""
    from tqllm_b200 import moe
    n, k, e, h = 17, 3, 6, 72
    ids, x, w, _, g = make(n, h, e, k, BF16, 4, skip=0.3)
    wide = lambda m: torch.full((m, 96), 3.0, dtype=BF16, device="cuda")
    xs, rs, ys, os_, gs, ds = wide(n), wide(n * k), wide(n * k), wide(n), wide(n * k), wide(n)
    view = lambda t, at=16: t[:, at:at + h]
    view(xs).copy_(x)
    plan = moe.dispatch(ids.cuda(), e)
    rows, slots = moe.dispatch_rows(view(xs), ids.cuda(), plan, rows=view(rs, 8))
    want, token = sorted_plain(ids, e, False)
    live = token.numel()
    assert torch.equal(view(rs, 8)[:live].cpu(), x[token]) and bool((rs[:, :8] == 3).all()) and bool((rs[:, 80:] == 3).all()) and bool((rs[live:] == 3).all())
    y, r = torch.randn(n * k, h, generator=g).to(BF16), torch.randn(n, h, generator=g).to(BF16)
    view(ys).copy_(y)
    view(os_, 0).copy_(r)
    out = moe.combine_rows(view(ys), slots, w.cuda(), n, k, residual=view(os_, 0), out=view(os_, 0))
    total, size = plain_back(y, want, w, None, r, n, k, False)
    near(out, total, (k + 3) * U * size, BF16)
    assert bool((os_[:, h:] == 3).all())
    view(ds).copy_(r)
    gy, gw, _ = moe.combine_rows_backward(view(ds), view(ys), slots, w.cuda(), n, k, grad_y=view(gs, 24))
    gy2, gw2, _ = moe.combine_rows_backward(r.cuda(), y.cuda(), slots, w.cuda(), n, k)
    assert torch.equal(gw, gw2) and torch.equal(gy[:live], gy2[:live]) and bool((gs[:, :24] == 3).all()) and bool((gs[live:] == 3).all())


def test_offsets_beyond_32_bits():
    from tqllm_b200 import moe
    n, k, e, h, ld = 2, 1, 2, 64, (1 << 32) + 64
    buf = torch.zeros(ld + h, dtype=BF16, device="cuda")
    far = buf.as_strided((n, h), (ld, 1))
    ids = torch.tensor([[1], [0]], dtype=torch.int32).cuda()
    x = torch.randn(n, h).to(BF16).cuda()
    far.copy_(x)
    plan = moe.dispatch(ids, e)
    rows, slots = moe.dispatch_rows(far, ids, plan)
    assert torch.equal(rows, x.flip(0)) and slots.tolist() == [1, 0]
    moe.dispatch_rows(x, ids, plan, rows=far)
    assert torch.equal(far, x.flip(0))
    assert torch.equal(moe.combine_rows(far, slots, None, n, k), x)
    moe.combine_rows(rows, slots, None, n, k, out=far)
    assert torch.equal(far, x)
    gy, gw, _ = moe.combine_rows_backward(far, rows, slots, None, n, k, grad_y=torch.zeros_like(rows))
    assert torch.equal(gy, x.flip(0))
    gy, gw2, _ = moe.combine_rows_backward(x, far, slots, None, n, k, grad_y=far)
    assert torch.equal(far, x.flip(0))


def test_captured():
    from tqllm_b200 import moe
    n, k, e, h = 12, 3, 8, 256
    ids, x, w, sw, g = make(n, h, e, k, BF16, 2)
    di, dx, dw, dsw = ids.cuda(), x.cuda(), w.cuda(), sw.cuda()

    def step():
        plan = moe.dispatch(di, e, n)
        rows, slots = moe.dispatch_rows(dx, di, plan)
        out = moe.combine_rows(rows, slots, dw, n, k, shared_weights=dsw)
        return rows, slots, out, moe.combine_rows_backward(out, rows, slots, dw, n, k, shared_weights=dsw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for seed in (3, 4):
        a, b, c, d, _ = make(n, h, e, k, BF16, seed, skip=0.25)
        for t, s in ((di, a), (dx, b), (dw, c), (dsw, d)):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        want, token = sorted_plain(a, e, True)
        assert torch.equal(got[1].cpu(), want) and torch.equal(got[0][: token.numel()].cpu(), b[token])
        total, size = plain_back(got[0].cpu(), want, c, d, None, n, k, True)
        near(got[2], total, (k + 3) * U * size, BF16)
        eager = moe.combine_rows_backward(got[2], got[0], got[1], dw, n, k, shared_weights=dsw)
        assert all(torch.equal(p, q) for p, q in zip(eager[1:], got[3][1:])) and torch.equal(eager[0][: token.numel()], got[3][0][: token.numel()])
