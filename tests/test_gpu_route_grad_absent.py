"""GPU: the gradient of normalised sigmoid weights where ids were set to no expert after the routing: what the routing divided by counts with every expert it selected.

Bound as in test_gpu_route_grad, against autograd of the whole selection: the weights' own roundings come in, (topk + 60) u of the terms, so 100 u of them."""
import pytest
import torch

from test_gpu_route_grad import CLAMP, U, routed

pytestmark = pytest.mark.gpu


def check(logits, e, k, scale, absent, g, norm=True):
    """absent [n, k]: assignments whose id becomes -1 (and one beyond the experts) behind the routing"""
    from tqllm_b200 import moe
    ids, w, _ = routed(logits, e, k, 2, norm, scale)
    marked = torch.where(absent, torch.where(torch.arange(k) % 2 == 0, -1, e), ids).to(torch.int32)
    got = moe.route_backward(logits.cuda(), marked.cuda(), w.cuda(), g.cuda(), e, 2, norm, scale).cpu().double()
    x = logits.double().requires_grad_()
    p = torch.sigmoid(x).gather(1, ids.long())
    total = p.sum(-1, keepdim=True)
    v = p / total.clamp(min=CLAMP) if norm else p
    factor = scale or 1.0
    want, = torch.autograd.grad((v * factor * g.double()).sum(), x)
    gone = torch.zeros(logits.shape, dtype=torch.bool).scatter_(1, ids.long(), absent)
    want = want.masked_fill(gone, 0.0)
    p, v = p.detach(), v.detach() * factor
    v = v.abs()                                                        # sizes of the terms, of a scale below zero too
    factor = abs(factor)
    size = v * ((v / factor)[:, None, :] * (g.double()[:, :, None] - g.double()[:, None, :]).abs()).sum(-1) + v * (v / factor * g.double().abs()).sum(-1, keepdim=True) + v * g.double().abs()
    room = torch.zeros_like(want).scatter_(1, ids.long(), 100 * U * size) + 2.0 ** -149
    bad = ~((got - want).abs() <= room)
    assert not bool(bad.any()), f"{got[bad][:4]} {want[bad][:4]} {room[bad][:4]}"


@pytest.mark.parametrize("scale", (0.0, 2.5, -1.0))
def test_the_large_one_is_elsewhere(scale):
    """the rest's sum is below the clamp, the whole selection's far above"""
    logits = torch.full((5, 16), -30.0) + 0.1 * torch.arange(16)
    logits[0, 3], logits[1, 9], logits[2, 0], logits[3, :4], logits[4] = 4.0, -1.0, 12.0, -8.0, -13.0 + 0.05 * torch.arange(16)
    g = torch.randn(5, 5, generator=torch.Generator().manual_seed(1))
    ids, _, _ = routed(logits, 16, 5, 2, True, scale)
    total = torch.sigmoid(logits.double()).gather(1, ids.long()).sum(-1)
    assert [bool(t > CLAMP) for t in total] == [True, True, True, True, False]
    absent = torch.zeros(5, 5, dtype=torch.bool)
    absent[:, 0] = True                                                # the largest of the selection comes first
    absent[3, :4] = True
    check(logits, 16, 5, scale, absent, g)


@pytest.mark.parametrize("k", (3, 40))
def test_any_selection(k):
    gen = torch.Generator().manual_seed(k)
    logits = torch.randn(300, 64, generator=gen) * 3 - torch.linspace(0, 25, 300)[:, None]
    g, absent = torch.randn(300, k, generator=gen), torch.rand(300, k, generator=gen) < 0.5
    ids, _, _ = routed(logits, 64, k, 2, True, 0.0)
    total = torch.sigmoid(logits.double()).gather(1, ids.long()).sum(-1)
    assert not bool(((total / CLAMP - 1).abs() < 1e-4).any())          # none so close that roundings decide
    check(logits, 64, k, 1.5, absent, g)
    check(logits, 64, k, 1.5, absent, g, norm=False)
