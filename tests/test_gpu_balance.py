"""GPU: the balance loss, its counts and its gradient against 64-bit arithmetic (autograd of the definition and differences).

Bound, relative to the size of the terms: a score is exp(l - max) or a sigmoid over a sum. The exponent's rounding gives |l - max| 2^-24 (l itself for
a sigmoid), exp 2 units, the sum over at most 4096 scores (32 a lane, then trees of 5 and 2 steps) 40, quotient and product 3: (48 + R) 2^-24 with
R = the largest |l - max| of a score that is not below e^-80 of the largest (the others are below the bound on the sum). The mean over tokens: 16 rows a warp, eight
warps, then the chunks (at most n / 8 of them, an eighth in turn) and 8: 40 + n / 64 roundings. So C = (100 + R + n / 64) 2^-24 for means and loss, and
C p (c + dot) factor for a gradient's entry, where c - dot is a difference of two such values."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(logits, ids, e, coef, gating, mask=None, offsets=None):
    """loss (differentiable in the 64-bit logits), counts, means, tokens"""
    n, k = ids.shape
    off = [0, n] if offsets is None else offsets.tolist()
    keep = torch.ones(n, dtype=torch.bool) if mask is None else mask.bool()
    u = logits[:, :e].double()
    if gating == 2:
        u = torch.nn.functional.logsigmoid(u)
    loss, counts, means, tokens = torch.zeros((), dtype=torch.float64), [], [], []
    spans = [torch.tensor([t for t in range(a, b) if keep[t]], dtype=torch.long) for a, b in zip(off, off[1:])]
    filled = sum(len(t) > 0 for t in spans)
    for t in spans:
        c = torch.zeros(e, dtype=torch.float64)
        for i in ids[t].flatten().tolist():
            if 0 <= i < e:
                c[i] += 1
        p = torch.softmax(u[t], -1)
        p = torch.where(torch.isneginf(u[t]).all(-1, keepdim=True), torch.zeros_like(p), p)
        mean = p.sum(0) / max(len(t), 1)
        counts.append(c)
        means.append(mean)
        tokens.append(len(t))
        if len(t):
            loss = loss + coef / filled * e / (k * len(t)) * (c * mean).sum()
    return loss, torch.stack(counts), torch.stack(means), tokens + [filled], p


def run(logits, ids, e, coef, gating, mask=None, offsets=None, **more):
    from tqllm_b200 import moe
    up = lambda t: None if t is None else t.cuda()
    l = logits.cuda()
    b = moe.balance_loss(l, up(ids), e, coef, gating, up(mask), up(offsets))
    g = moe.balance_loss_backward(l, b, ids.shape[1], coef, gating, up(mask), up(offsets), **more)
    return b, g


def make(n, e, k, seed, scale=2.0, ld=None):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(n, ld or e, generator=g) * scale
    ids = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(n)]).int()
    return logits, ids, g


def check(logits, ids, e, coef, gating, mask=None, offsets=None, grad_scale=1.0, b=None, grad=None):
    n = ids.shape[0]
    live = torch.nan_to_num(logits[:, :e], nan=0.0, neginf=0.0)
    spread = float(min(80.0, 2 * live.abs().max()))
    C = (100 + spread + n / 64) * 2.0 ** -24
    x = logits.double().requires_grad_()
    loss, counts, means, tokens, _ = plain(x, ids, e, coef, gating, mask, offsets)
    assert torch.equal(b.counts.cpu().double(), counts) and b.tokens.tolist() == tokens
    assert bool(((b.prob.cpu().double() - means).abs() <= C * means + 1e-36).all())
    assert abs(float(b.loss) - float(loss.detach())) <= C * abs(float(loss.detach())) + 1e-36
    want, = torch.autograd.grad(loss * grad_scale, x) if loss.requires_grad else (torch.zeros_like(x),)
    want = torch.nan_to_num(want[:, :e].detach(), nan=0.0)
    # the size of what is subtracted: p (c + dot) factor, from the gradient of the definition with its parts
    off = [0, n] if offsets is None else offsets.tolist()
    size = torch.zeros(n, e, dtype=torch.float64)
    for s, (a, z) in enumerate(zip(off, off[1:])):
        if tokens[s]:
            u = logits[a:z, :e].double()
            p = torch.softmax(torch.nn.functional.logsigmoid(u) if gating == 2 else u, -1)
            f = abs(grad_scale) * coef / tokens[-1] * e / (ids.shape[1] * tokens[s] ** 2)
            size[a:z] = torch.nan_to_num(p) * (counts[s] + torch.nan_to_num(p) @ counts[s][:, None]) * f
    got = grad[:, :e].cpu().double()
    keep = torch.ones(n, dtype=torch.bool) if mask is None else mask.bool()
    keep = keep & (torch.arange(n) >= off[0]) & (torch.arange(n) < off[-1])
    assert bool((got[~keep] == 0).all())
    assert bool(((got - want).abs() <= C * size + 1e-36)[keep].all())


@pytest.mark.parametrize("e,k", ((1, 1), (2, 1), (31, 4), (32, 2), (33, 8), (64, 6), (100, 3), (128, 8), (200, 10), (300, 4), (512, 10), (513, 2), (1000, 8), (1025, 4), (2049, 3), (4096, 10)))
@pytest.mark.parametrize("gating", (1, 2))
def test_experts(e, k, gating):
    n = 37
    logits, ids, _ = make(n, e, k, e + k)
    b, g = run(logits, ids, e, 0.01, gating)
    check(logits, ids, e, 0.01, gating, b=b, grad=g)


@pytest.mark.parametrize("n", (1, 2, 7, 8, 9, 64, 65, 300, 2369, 5000))
@pytest.mark.parametrize("gating", (1, 2))
def test_tokens(n, gating):
    logits, ids, _ = make(n, 60, 6, n)
    b, g = run(logits, ids, 60, 0.5, gating)
    check(logits, ids, 60, 0.5, gating, b=b, grad=g)


@pytest.mark.parametrize("gating", (1, 2))
@pytest.mark.parametrize("e", (48, 700))
def test_sequences_and_masks(gating, e):
    """ragged and empty sequences, rows in front and behind, a sequence that the mask empties, ids that are skipped, poison in masked rows"""
    n = 203
    logits, ids, gen = make(n, e, 4, 5, ld=e + 1)
    offsets = torch.tensor([3, 3, 4, 50, 50, 130, 131, 190, 190], dtype=torch.int32)
    mask = torch.rand(n, generator=gen) < 0.7
    mask[130] = False                                                  # the sequence of one token
    logits[~mask] = float("nan")
    logits[:3], logits[190:] = float("inf"), float("nan")
    ids[torch.rand(n, 4, generator=gen) < 0.2] = -1
    ids[60, 1] = e
    ids[~mask] = 0
    b, g = run(logits, ids, e, 0.01, gating, mask, offsets)
    check(torch.nan_to_num(logits, nan=0.0, posinf=0.0), ids, e, 0.01, gating, mask, offsets, b=b, grad=g)
    assert bool(torch.isfinite(g).all())


@pytest.mark.parametrize("n", (1, 33, 64, 65))
@pytest.mark.parametrize("e", (40, 600, 2048, 2049))
@pytest.mark.parametrize("span", ((0, None), (1, None), (5, 30), (64, 64), (0, 0)))
def test_one_sequence_of_a_few_tokens(n, e, span):
    """with rows in front and behind, a mask, nothing at all"""
    logits, ids, gen = make(n, e, 3, n + e)
    a, z = min(span[0], n), n if span[1] is None else min(span[1], n)
    offsets = torch.tensor([a, max(a, z)], dtype=torch.int32)
    for mask in (None, torch.rand(n, generator=gen) < 0.6):
        b, g = run(logits, ids, e, 0.1, 1, mask, offsets)
        check(logits, ids, e, 0.1, 1, mask, offsets, b=b, grad=g)


@pytest.mark.parametrize("e", (40, 600))
def test_nothing_left(e):
    from tqllm_b200 import moe
    logits, ids, _ = make(30, e, 2, 1)
    b, g = run(logits, ids, e, 0.1, 1, mask=torch.zeros(30, dtype=torch.bool))
    assert float(b.loss) == 0.0 and not bool(b.counts.any()) and not bool(b.prob.any()) and b.tokens.tolist() == [0, 0] and not bool(g.any())
    b, g = run(logits, torch.full_like(ids, -1), e, 0.1, 1)
    assert float(b.loss) == 0.0 and b.tokens.tolist() == [30, 1] and not bool(g.any())


@pytest.mark.parametrize("gating", (1, 2))
@pytest.mark.parametrize("e", (40, 600))
def test_masked_logits_and_infinities(gating, e):
    """-inf and the lowest value of the type as an expert mask, a row that has nothing else, values that overflow an exponential; then a NaN"""
    logits, ids, _ = make(20, e, 3, 2)
    logits[:, 5] = float("-inf")
    logits[:, 6] = torch.finfo(torch.float32).min
    logits[3] = float("-inf")
    logits[4] = -1e4
    logits[4, 7] = -9990.0
    logits[5] = 1e4
    logits[6] *= 40
    logits[7] = -90.0 + logits[7]
    b, g = run(logits, ids, e, 0.1, gating)
    x = logits.clone()
    check(x, ids, e, 0.1, gating, b=b, grad=g)
    assert bool((g[3] == 0).all()) and bool(torch.isfinite(g).all()) and bool(torch.isfinite(b.loss))
    logits[9, 1] = float("nan")
    b, g = run(logits, ids, e, 0.1, gating)
    assert bool(torch.isnan(b.loss)) and bool(torch.isnan(g[9]).all()) and int(torch.isnan(g).any(-1).sum()) == 1
    assert torch.equal(b.counts.cpu().flatten().long(), torch.bincount(ids.flatten().long(), minlength=e))


@pytest.mark.parametrize("e", (50, 900))
def test_added_to_a_gradient(e):
    logits, ids, gen = make(70, e, 4, 3, ld=e + 3)
    mask = torch.rand(70, generator=gen) < 0.5
    have = torch.randn(70, e + 2, generator=gen)
    out = have.cuda()
    scale = torch.tensor(-3.0)
    b, alone = run(logits, ids, e, 0.2, 1, mask, grad_loss=scale.cuda())
    check(logits, ids, e, 0.2, 1, mask, grad_scale=-3.0, b=b, grad=alone)
    run(logits, ids, e, 0.2, 1, mask, grad_loss=scale.cuda(), out=out)
    got = out.cpu()
    assert torch.equal(got[:, e:], have[:, e:]) and torch.equal(got[~mask], have[~mask])
    assert torch.equal(got[:, :e], have[:, :e] + alone.cpu())


def test_gradient_against_differences():
    """central differences of the 64-bit definition: the device's gradient and autograd both"""
    for gating in (1, 2):
        logits, ids, _ = make(12, 9, 2, 4)
        offsets = torch.tensor([0, 5, 12], dtype=torch.int32)
        b, g = run(logits, ids, 9, 1.0, gating, offsets=offsets)
        f = lambda x: float(plain(x, ids, 9, 1.0, gating, offsets=offsets)[0])
        for t in range(12):
            for j in range(9):
                d = torch.zeros(12, 9, dtype=torch.float64)
                d[t, j] = 1e-4
                slope = (f(logits.double() + d) - f(logits.double() - d)) / 2e-4
                assert abs(float(g[t, j]) - slope) <= 1e-6 * abs(slope) + 1e-8       # third derivative x 1e-8 / 6, and 2^-24 x 100


def test_the_same_bits_every_time_on_streams_and_in_graphs():
    from tqllm_b200 import moe
    logits, ids, _ = make(3000, 130, 8, 6)
    l, i = logits.cuda(), ids.cuda()
    offsets = torch.tensor([0, 1000, 1007, 3000], dtype=torch.int32, device="cuda")
    call = lambda: (lambda b: (*b, moe.balance_loss_backward(l, b, 8, 0.1, offsets=offsets)))(moe.balance_loss(l, i, 130, 0.1, offsets=offsets))
    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = call()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    l.mul_(-0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, call()))


def test_counts_place_experts():
    """the counts of a routed batch feed the placement like a histogram of its ids"""
    from tqllm_b200 import moe
    logits, _, _ = make(400, 32, 4, 7, ld=33)
    l = logits.cuda()
    ids, _, _ = moe.topk_softmax(l, 32, 4)
    b = moe.balance_loss(l, ids, 32, 0.01)
    hist = moe.count_ids(ids, torch.zeros(32, dtype=torch.int64, device="cuda"))
    assert torch.equal(b.counts[0].long(), hist)
    assert torch.equal(torch.from_numpy(moe.place_experts(b.counts[0], 4)[0]), torch.from_numpy(moe.place_experts(hist, 4)[0]))


@pytest.mark.parametrize("e,k,n", ((1, 1, 5), (6, 6, 70), (40, 40, 9), (700, 7, 100), (64, 8, 4000), (2100, 3, 700)))
@pytest.mark.parametrize("gating", (1, 2))
def test_an_even_load_has_no_gradient(e, k, n, gating):
    """equal counts: c - sum p c is zero whatever p is, and no rounding of the sum is left in its place"""
    logits, _, _ = make(n, e, k, e)
    ids = (torch.arange(n * k) % e).view(n, k).int()
    assert n * k % e == 0
    b, g = run(logits, ids, e, 3.0, gating)
    assert torch.equal(b.counts.cpu(), torch.full((1, e), n * k // e, dtype=torch.int32))
    assert not bool(g.any())


@pytest.mark.parametrize("e", (60, 700))
@pytest.mark.parametrize("gating", (1, 2))
def test_a_nearly_even_load(e, gating):
    """Counts of 1,000 (or 200) and a few: the error is relative to what they have more than the least, which is little of them. Scores are sums of positive numbers: the bound of the definition, C as above."""
    k, coef = 5, 1.0
    n = (1000 if e == 60 else 200) * e // k
    logits, _, gen = make(300, e, k, e)
    logits = logits.repeat(-(-n // 300), 1)[:n]
    ids = (torch.arange(n * k) % e).view(n, k).int()
    ids[:40, 0] = torch.randint(0, e // 2, (40,), generator=gen).int()
    b, g = run(logits, ids, e, coef, gating)
    c = torch.bincount(ids.flatten().long(), minlength=e).double()
    assert torch.equal(b.counts[0].cpu().double(), c)
    x = c - c.min()
    u = logits.double()
    p = torch.softmax(torch.nn.functional.logsigmoid(u) if gating == 2 else u, -1)
    f = coef * e / (k * float(n) ** 2) * (torch.sigmoid(-u) if gating == 2 else 1.0)
    want, size = p * (x - p @ x[:, None]) * f, p * (x + p @ x[:, None]) * f
    C = (100 + float(2 * logits.abs().max())) * 2.0 ** -24
    assert bool(((g.cpu().double() - want).abs() <= C * size + 1e-36).all())
