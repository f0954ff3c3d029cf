"""GPU: the norm's gradient where the sum of gradients times rows passes 32 bits and neither the squares nor the gradient do, through every form."""
import pytest
import torch

from test_gpu_norm import BF16, F32
from test_gpu_norm_gradient_far import EPS, FORMS, check, make, place

pytestmark = pytest.mark.gpu
LARGE = ((1.0, 1e-2), (1e14, 1e25), (1e3, 1e36), (1e18, 1e30), (1e30, 1e30), (1e30, 1e5), (1e-25, 1e12), (1e-3, 1e33))


@pytest.mark.parametrize("form,n,k", FORMS)
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", (0.0, EPS))
def test_sums_beyond_32_bits(form, n, k, dtype, eps):
    from tqllm_b200 import moe
    h, w, g, s = make(n, k, dtype, LARGE, n + k)
    g[1::2] = g[1::2].abs() * h[1::2].float().sign().to(dtype)         # all products of one sign: the sums pass the range, the gradient does not
    got, weight = moe.rms_norm_backward(place(h, form, False), w.cuda(), place(g, form, False), eps, place(s, form, False), out=place(torch.zeros_like(h), form, True))
    check(h, w, g, s, eps, got, weight, dtype, form)


@pytest.mark.parametrize("form,n,k", FORMS)
def test_what_is_not_finite_stays_in_its_row(form, n, k):
    from tqllm_b200 import moe
    h, w, g, s = make(n, k, F32, LARGE, n + k)
    h[2, k // 2], g[5, k - 1], h[8, 0] = float("nan"), float("inf"), float("-inf")
    got, none = moe.rms_norm_backward(place(h, form, False), w.cuda(), place(g, form, False), EPS, place(s, form, False), out=place(torch.zeros_like(h), form, True), weight_grad=False)
    assert none is None
    got, keep = got.cpu(), [i for i in range(n) if i not in (2, 5, 8)]
    assert bool(got[2].isnan().all()) and not got[5].isfinite().any() and not got[8].isfinite().all()
    check(h[keep], w, g[keep], s[keep], EPS, got[keep], None, F32, form)
