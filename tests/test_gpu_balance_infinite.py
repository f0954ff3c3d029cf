"""GPU: logits of +inf in the balance loss. The softmax's difference of two infinities is a NaN, which stays in its row and shows in the loss; a sigmoid of it is one. Bound as in the tests of the
loss: (100 + R) 2^-24 of p (c + sum p c) times the factor, R the largest finite logit's size."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e", (40, 600))
@pytest.mark.parametrize("n", (20, 300))
def test_plus_infinity(e, n):
    from tqllm_b200 import moe
    g = torch.Generator().manual_seed(e + n)
    logits, ids = torch.randn(n, e, generator=g), torch.randint(0, e, (n, 3), generator=g, dtype=torch.int32).cuda()
    logits[4, 7] = logits[9, 0] = logits[9, e - 1] = float("inf")
    l = logits.cuda()
    b = moe.balance_loss(l, ids, e, 0.1)
    grad = moe.balance_loss_backward(l, b, 3, 0.1)
    assert bool(torch.isnan(b.loss)) and bool(torch.isnan(grad[[4, 9]]).all()) and int(torch.isnan(grad).any(-1).sum()) == 2
    b = moe.balance_loss(l, ids, e, 0.1, gating=2)
    grad = moe.balance_loss_backward(l, b, 3, 0.1, gating=2).double()
    s = torch.sigmoid(l.double())
    p = s / s.sum(-1, keepdim=True)
    c = torch.bincount(ids.flatten().long(), minlength=e).double()
    C = (100 + float(logits[torch.isfinite(logits)].abs().max())) * 2.0 ** -24
    f = 0.1 * e / (3 * float(n) ** 2) * (1.0 - s)
    assert bool(((b.prob[0].double() - p.mean(0)).abs() <= (C + n / 64 * 2.0 ** -24) * p.mean(0)).all())
    assert bool(((grad - p * (c - p @ c[:, None]) * f).abs() <= C * p * (c + p @ c[:, None]) * f + 1e-36).all())
    assert bool((grad[l.isinf()] == 0).all())
