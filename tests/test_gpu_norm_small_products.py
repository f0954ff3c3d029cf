"""GPU: rows to 8 bits whose products with the weight lie below the normal numbers of 32 bits: integers and scales are those of the products as they are before any rounding.

The scale's bound is that of rows of an ordinary size, 27 u and the smallest number."""
import pytest
import torch

from test_gpu_norm import BF16, F32, U, integers
from test_gpu_norm_small_squares import WHOLE, check, far_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,k", ((6, 16), (6, 512), (2400, 256), (2400, 2048), (6, 16384)))
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", (0.0, 1e-30, 1e-17, 1e-6))
@pytest.mark.parametrize("size,weight", ((2.0 ** -100, 2.0 ** -40), (2.0 ** -80, 2.0 ** -60), (2.0 ** -126, 1.0), (2.0 ** -126, 2.0 ** -100), (1.0, 2.0 ** -126)))
def test_products_below_the_normal_numbers(n, k, dtype, eps, size, weight):
    from tqllm_b200 import moe
    g = torch.Generator().manual_seed(k)
    x, w = (torch.randn(n, k, generator=g) * size).to(dtype), torch.rand(k, generator=g) * weight + weight
    x[1] = 0
    out = moe.rms_norm(x.cuda(), w.cuda(), eps, rows=False, quantize=True)
    h = x.double()
    u, root = h * w.double(), (h.square().mean(-1) + float(torch.tensor(eps, dtype=F32))).sqrt()
    top = u.abs().amax(-1)
    assert torch.equal(out.q.cpu().double(), integers(u))
    want = torch.where(top > 0, top / root / 127, torch.zeros_like(top))
    bad = ~((out.scale.cpu().double() - want).abs() <= 27 * U * want + 2.0 ** -149)
    assert not bool(bad.any()), f"{out.scale.cpu()[bad][:4]} {want[bad][:4]}"


@pytest.mark.parametrize("n,k", WHOLE)
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", (0.0, 1e-25))
def test_rows_of_all_sizes(n, k, dtype, eps):
    from tqllm_b200 import moe
    x, w = far_rows(n, k, dtype, n), 1 + 0.1 * torch.randn(k, generator=torch.Generator().manual_seed(k))
    check(x, None, w, eps, moe.rms_norm(x.cuda(), w.cuda(), eps, quantize=True), dtype, 0.0)
