"""GPU: small rows with every small eps, those beside the border below which a row is looked at again among them. Bounds as for rows of an ordinary size."""
import pytest
import torch

from test_gpu_norm import BF16, F32
from test_gpu_norm_gradient_far import SMALL, make, place
from test_gpu_norm_gradient_far import check as check_gradient
from test_gpu_norm_small_squares import check, far_rows

pytestmark = pytest.mark.gpu
EPS = (2.0 ** -64, 2.0 ** -64 * (1 - 2.0 ** -24), 2.0 ** -63, 1e-20, 1e-21, 1e-23, 1e-28, 1e-33, 2.0 ** -126, 2.0 ** -149)


@pytest.mark.parametrize("n,k", ((19, 64), (38, 1024), (2375, 512), (2375, 2064), (38, 8208), (38, 65), (57, 4097)))
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", EPS)
def test_norm(n, k, dtype, eps):
    from tqllm_b200 import moe
    x, w = far_rows(n, k, dtype, n + k), 1 + 0.1 * torch.randn(k, generator=torch.Generator().manual_seed(k))
    check(x, None, w, eps, moe.rms_norm(x.cuda(), w.cuda(), eps, quantize=k % 16 == 0), dtype, 0.0)


@pytest.mark.parametrize("form,n,k", (("whole", 40, 64), ("whole", 300, 2048), ("whole", 30, 16384), ("shifted", 40, 61), ("shifted", 300, 2047), ("single", 40, 64), ("single", 30, 4093)))
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", EPS)
def test_gradient(form, n, k, dtype, eps):
    from tqllm_b200 import moe
    h, w, g, s = make(n, k, dtype, SMALL + ((1e-10, 1e25), (0.0, 1e-3)), n + k)
    got, weight = moe.rms_norm_backward(place(h, form, False), w.cuda(), place(g, form, False), eps, place(s, form, False), out=place(torch.zeros_like(h), form, True))
    check_gradient(h, w, g, s, eps, got, weight, dtype, form)
