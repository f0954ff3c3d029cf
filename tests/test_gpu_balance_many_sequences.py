"""GPU: the balance loss over thousands of sequences, empty ones among them, up to as many as a call takes, against 64-bit sums. A sequence has at most 40 tokens here: bounds as in the tests of the
loss, without their term for long means: C = (100 + R) 2^-24, R the largest distance of two logits of a row."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences,most,e", ((1000, 40, 8), (5000, 3, 33), (20000, 1, 16), (65535, 2, 4), (300, 7, 600)))
@pytest.mark.parametrize("masked", (False, True))
def test_many(sequences, most, e, masked):
    from tqllm_b200 import moe
    g = torch.Generator().manual_seed(sequences)
    lengths = torch.randint(0, most + 1, (sequences,), generator=g)
    lengths[sequences // 2: sequences // 2 + 90] = 0                   # a run of empty ones
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), lengths.cumsum(0)]) + 2
    n, k, coef = int(offsets[-1]) + 3, 2, 0.7                          # rows in front of the first and behind the last
    logits = torch.randn(n, e, generator=g).cuda()
    ids = torch.randint(0, e, (n, k), generator=g, dtype=torch.int32).cuda()
    mask = (torch.rand(n, generator=g) < 0.6).cuda() if masked else None
    off = offsets.int().cuda()
    b = moe.balance_loss(logits, ids, e, coef, mask=mask, offsets=off)
    grad = moe.balance_loss_backward(logits, b, k, coef, mask=mask, offsets=off).double()
    of = torch.repeat_interleave(torch.arange(sequences), lengths).cuda()
    at = torch.arange(2, n - 3).cuda()
    if masked:
        of, at = of[mask[at]], at[mask[at]]
    p = torch.softmax(logits[at].double(), -1)
    tokens = torch.zeros(sequences, dtype=torch.long, device="cuda").index_add_(0, of, torch.ones_like(of))
    counts = torch.zeros(sequences * e, dtype=torch.long, device="cuda")
    counts.index_add_(0, (of[:, None] * e + ids[at]).flatten(), torch.ones(at.numel() * k, dtype=torch.long, device="cuda"))
    counts, filled = counts.view(sequences, e), int((tokens > 0).sum())
    assert torch.equal(b.counts.long(), counts) and torch.equal(b.tokens[:-1].long(), tokens) and int(b.tokens[-1]) == filled
    per = tokens.clamp(min=1).double()[:, None]
    mean = torch.zeros(sequences, e, dtype=torch.float64, device="cuda").index_add_(0, of, p) / per
    C = (100 + float(logits.max() - logits.min())) * 2.0 ** -24
    assert bool(((b.prob.double() - mean).abs() <= C * mean).all())
    factor = coef * e / k / filled
    loss = float((factor * (counts * mean).sum(-1) / per[:, 0]).sum())
    assert abs(float(b.loss) - loss) <= C * loss
    x = (counts - counts.amin(-1, keepdim=True)).double()[of]
    f = factor / per[of] ** 2
    dot = (p * x).sum(-1, keepdim=True)
    want, size = torch.zeros_like(grad), torch.zeros_like(grad)
    want[at], size[at] = p * (x - dot) * f, p * (x + dot) * f
    assert bool(((grad - want).abs() <= 2 * C * size).all())
