"""GPU: eps above one and up to the end of 32 bits, with rows and gradients whose sums pass the range. Bounds as for rows of an ordinary size."""
import pytest
import torch

from test_gpu_norm import BF16, F32
from test_gpu_norm_gradient_far import check as check_gradient
from test_gpu_norm_gradient_far import make, place
from test_gpu_norm_gradient_large_sums import LARGE
from test_gpu_norm_small_squares import check

pytestmark = pytest.mark.gpu
EPS = (1.0, 20.0, 1e4, 1e12, 1e25, 3e38)


@pytest.mark.parametrize("form,n,k", (("whole", 40, 64), ("whole", 300, 2048), ("whole", 30, 16384), ("shifted", 40, 61), ("shifted", 300, 2047), ("single", 40, 64), ("single", 30, 4093)))
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", EPS)
def test_gradient(form, n, k, dtype, eps):
    from tqllm_b200 import moe
    h, w, g, s = make(n, k, dtype, LARGE + ((1.0, 1e37), (1e-3, 3e37)), n + k)
    g[1::2] = g[1::2].abs() * h[1::2].float().sign().to(dtype)         # all products of one sign
    got, weight = moe.rms_norm_backward(place(h, form, False), w.cuda(), place(g, form, False), eps, place(s, form, False), out=place(torch.zeros_like(h), form, True))
    check_gradient(h, w, g, s, eps, got, weight, dtype, form)


@pytest.mark.parametrize("n,k", ((19, 64), (2375, 512), (38, 8208), (38, 65), (57, 4097)))
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", EPS)
def test_norm(n, k, dtype, eps):
    from tqllm_b200 import moe
    h, w, _, _ = make(n, k, dtype, ((1.0, 1.0), (1e10, 1.0), (1e19, 1.0), (1e20, 1.0), (1e30, 1.0), (5e37, 1.0)), n + k)
    check(h, None, w, eps, moe.rms_norm(h.cuda(), w.cuda(), eps, quantize=k % 16 == 0), dtype, 0.0)
