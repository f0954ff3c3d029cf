"""GPU: the gradient of the balance loss from counts that 32-bit floats do not hold: what an expert has more than the least is a difference of whole numbers. The counts and tokens are made by hand (a
batch of that many tokens is not needed: the gradient takes them from the loss, or from a sum over ranks).

Bound, in units of 2^-24: a score p is off by 48 + R (the header of the loss's tests derives it; R: the largest distance of a logit from the row's largest, or its size for a sigmoid), the sum of p x
over the experts by 48 + R and 41 more, x = c - min c by one (a whole number below 2^30), the slope of a sigmoid by 5, products and the factor by 10. With x >= 0 every term is relative to p (x + sum p x)
times the factor: C = (160 + 2 R) 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e", (2, 33, 60, 512, 600, 2048, 4096))
@pytest.mark.parametrize("gating", (1, 2))
@pytest.mark.parametrize("base,more", ((0, 40), (1 << 24, 3), ((1 << 26) + 1, 7), ((1 << 29) + 5, 60), (3, 1 << 29)))
def test_counts_past_24_bits(e, gating, base, more):
    from tqllm_b200 import moe
    n, k, coef = 37, 2, 0.5
    g = torch.Generator().manual_seed(e + more)
    logits = torch.randn(n, e, generator=g) * 2
    counts = (base + torch.randint(0, more + 1, (1, e), generator=g)).int()
    tokens = torch.tensor([int(counts.sum(dtype=torch.int64)) // k % (1 << 30) + 1, 1], dtype=torch.int32)
    saved = moe.Balance(torch.zeros(()).cuda(), counts.cuda(), torch.zeros(1, e).cuda(), tokens.cuda())
    got = moe.balance_loss_backward(logits.cuda(), saved, k, coef, gating).cpu().double()
    x = (counts[0] - counts.min()).double()
    u = logits.double()
    p = torch.softmax(torch.nn.functional.logsigmoid(u) if gating == 2 else u, -1)
    f = coef * e / (k * float(tokens[0]) ** 2) * (torch.sigmoid(-u) if gating == 2 else 1.0)
    want, size = p * (x - p @ x[:, None]) * f, p * (x + p @ x[:, None]) * f
    C = (160 + 2 * float(2 * logits.abs().max())) * 2.0 ** -24
    assert bool(((got - want).abs() <= C * size + 1e-36).all())
