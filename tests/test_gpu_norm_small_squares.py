"""GPU: rows at the far ends of 32 bits through every form of the norm: squares that vanish or pass the range, with and without eps, zeros, infinities and NaN.

Bounds as for rows of an ordinary size: the unit that such a row is taken in is a power of two, so it adds no rounding."""
import pytest
import torch

from test_gpu_norm import BF16, F16, F32, U, integers, near

pytestmark = pytest.mark.gpu
LARGEST = float(torch.finfo(F32).max)


def far_rows(n, k, dtype, seed):
    """rows of sizes from the smallest values to the largest, repeated; none of them alike"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, k, generator=g)
    spread = torch.exp2(torch.randint(-60, 1, (n, k), generator=g).float())
    sizes = (1.0, 1e-12, 1e-19, 1e-20, 1e-23, 1e-30, 3e-38, 1e-39, 1e15, 1e18, 2e19, 1e30, 4e37)
    for i in range(n):
        case = i % (len(sizes) + 6)
        if case < len(sizes):
            x[i] = (x[i] * sizes[case]).clamp(-3e38, 3e38)
        elif case == len(sizes):
            x[i] = 0
        elif case == len(sizes) + 1:
            x[i] = 0
            x[i, k // 2] = 1e-44 if dtype is F32 else 1e-40                # one value, below the normal ones
        elif case == len(sizes) + 2:
            x[i] *= spread[i] * 1e-24
        elif case == len(sizes) + 3:
            x[i] *= spread[i]
            x[i, k - 1] = 2.0 ** 65                                    # values far below a row's largest keep their bits
        elif case == len(sizes) + 4:
            x[i, 0] = float("inf")
        else:
            x[i, k - 1] = float("nan")
    return x.to(dtype)


def root_of(h, eps):
    return (h.square().mean(-1, keepdim=True) + float(torch.tensor(eps, dtype=F32))).sqrt()


def check(x, r, w, eps, out, dtype, products=2.0 ** -100):
    """products: scales of rows whose largest product with the weight is at least this"""
    h = (x.float() if r is None else x.float() + r.float()).double()
    root = root_of(h, eps)
    if out.y is not None:
        y, want = out.y.cpu(), h / root * w.double()
        assert torch.equal(y.isnan(), want.isnan())
        fine = ~want.isnan()
        near(y[fine], want[fine], 26 * U * want[fine].abs(), dtype)
    if out.q is None:
        return
    u = h * w.double()
    fine = u.isfinite().all(-1) & (u.abs().amax(-1) <= LARGEST)
    q, scale = out.q.cpu(), out.scale.cpu()
    assert bool(scale[~fine].isnan().all()) and not q[~fine].any()
    assert torch.equal(q[fine].double(), integers(u[fine]))
    top = u[fine].abs().amax(-1)
    want = torch.where(top > 0, top / root[fine, 0] / 127, torch.zeros_like(top))
    bad = ~((scale[fine].double() - want).abs() <= 27 * U * want + 2.0 ** -149) & ((top == 0) | (top >= products))
    assert not bool(bad.any()), f"{scale[fine][bad][:4]} {want[bad][:4]}"


# a piece a thread; a warp a row; 128 threads; 512 threads
WHOLE = ((19, 16), (38, 1024), (57, 4096), (2375, 256), (2375, 1024), (2375, 2064), (38, 8208), (38, 16384))


@pytest.mark.parametrize("n,k", WHOLE)
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", (0.0, 1e-44, 1e-38, 1e-25, 1e-6))
def test_whole_rows(n, k, dtype, eps):
    from tqllm_b200 import moe
    x = far_rows(n, k, dtype, n + k)
    w = 1 + 0.1 * torch.randn(k, generator=torch.Generator().manual_seed(k))
    both = moe.rms_norm(x.cuda(), w.cuda(), eps, quantize=True)
    check(x, None, w, eps, both, dtype)
    plain = moe.rms_norm(x.cuda(), w.cuda(), eps)
    assert torch.equal(plain.y.view(torch.int16 if dtype is BF16 else torch.int32), both.y.view(torch.int16 if dtype is BF16 else torch.int32))
    only = moe.rms_norm(x.cuda(), w.cuda(), eps, rows=False, quantize=True)
    assert torch.equal(only.q, both.q) and torch.equal(only.scale.view(torch.int32), both.scale.view(torch.int32))


# blocks that walk rows, of a piece a thread and of several, and (another phase of the output) value by value
@pytest.mark.parametrize("n,k", ((38, 33), (1200, 1023), (2375, 1023), (700, 2049), (57, 8191), (399, 16383)))
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("eps", (0.0, 1e-38, 1e-6))
@pytest.mark.parametrize("single", (False, True))
def test_rows_that_begin_anywhere(n, k, dtype, eps, single):
    from tqllm_b200 import moe
    x = far_rows(n, k, dtype, n + k)
    w = 1 + 0.1 * torch.randn(k, generator=torch.Generator().manual_seed(k))
    out = torch.empty(n * k + 1, dtype=dtype, device="cuda")[int(single) : n * k + int(single)].view(n, k)
    check(x, None, w, eps, moe.rms_norm(x.cuda(), w.cuda(), eps, out=out), dtype)


@pytest.mark.parametrize("n,k", ((38, 512), (2375, 512), (38, 16384)))
def test_with_the_skip_connection_and_half_precision(n, k):
    """sums of two small rows; fp16, whose squares never leave 32 bits, and a weight of its own"""
    from tqllm_b200 import moe
    g = torch.Generator().manual_seed(k)
    w = 1 + 0.1 * torch.randn(k, generator=g)
    x, r = far_rows(n, k, BF16, 1), far_rows(n, k, BF16, 1)
    r = torch.where(r.isfinite(), -r * 0.5, r)
    out = moe.rms_norm(x.cuda(), w.cuda(), 0.0, r.cuda(), quantize=True)
    h = x.float() + r.float()
    assert torch.equal(out.sum.cpu().view(torch.int16), h.to(BF16).view(torch.int16)) or bool((out.sum.cpu().isnan() == h.isnan()).all())
    check(x, r, w, 0.0, out, BF16)
    x = (torch.randn(n, k, generator=g) * 6e-8).to(F16)
    x[::2] *= 1e4
    w = w.to(F16)
    check(x, None, w, 0.0, moe.rms_norm(x.cuda(), w.cuda(), 0.0, quantize=True), F16)


