"""GPU: the norm and its gradient onto their own inputs, with matrices that begin alike and with one that begins elsewhere: the same bits as into a buffer of their own."""
import pytest
import torch

from test_gpu_norm import BF16, F16, F32, check_norm, make
from test_gpu_norm_gradient_far import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("n,k,ld", ((19, 33, 48), (2500, 101, 101), (19, 1031, 1040), (301, 2050, 2051), (30, 8193, 8193), (19, 64, 64), (300, 512, 520)))
@pytest.mark.parametrize("lone", (None, 0, 1, 2))
def test_onto_the_inputs(dtype, n, k, ld, lone):
    """lone: the matrix that begins a value later than the others"""
    from tqllm_b200 import moe
    x, r, w, gen = make(n, k, dtype, F32, k + ld)
    g = torch.randn(n, k, generator=gen).to(dtype)

    def views(*values):
        out = [torch.full((n * ld + 16,), 3.0, dtype=dtype, device="cuda")[1 + (i == lone):].as_strided((n, k), (ld, 1)) for i in range(3)]
        for v, t in zip(out, values):
            v.copy_(t)
        return out
    form = "single" if lone is not None else "shifted"
    h, dy, ds = views(x, g, r)
    want, weight = moe.rms_norm_backward(h, w.cuda(), dy, 1e-6, ds, out=torch.empty(n * ld + 8, dtype=dtype, device="cuda")[1:].as_strided((n, k), (ld, 1)))
    check(x, w, g, r, 1e-6, want, weight, dtype, form)
    for i in range(3):
        place = views(x, g, r)
        got, same = moe.rms_norm_backward(place[0], w.cuda(), place[1], 1e-6, place[2], out=place[i])
        assert got.data_ptr() == place[i].data_ptr() and torch.equal(got, want) and torch.equal(same, weight)
    x1, r1, y1 = views(x, r, x)
    s1 = torch.empty(n * ld + 8, dtype=dtype, device="cuda")[1:].as_strided((n, k), (ld, 1))
    want = moe.rms_norm(x1, w.cuda(), 1e-6, r1, out=y1, sum_out=s1)
    check_norm(x, r, w, want, dtype)
    for y_on, sum_on in ((0, 1), (1, 0), (0, 2), (2, 0)):
        if lone == 2 and 2 not in (y_on, sum_on):
            continue                                                   # the matrix that begins elsewhere is not in the call
        place = views(x, r, x)
        got = moe.rms_norm(place[0], w.cuda(), 1e-6, place[1], out=place[y_on], sum_out=place[sum_on])
        assert torch.equal(got.y, want.y) and torch.equal(got.sum, want.sum)


@pytest.mark.parametrize("n,k,dtype", ((30011, 64, BF16), (30000, 256, BF16), (20000, 77, F16), (9001, 520, F32), (3001, 2056, BF16), (2003, 4099, F32), (1, 4096, BF16), (150, 16384, F32)))
def test_the_weights_gradient_within_its_own_steps(n, k, dtype):
    from tqllm_b200 import moe
    x, r, w, gen = make(n, k, dtype, F32, n)
    g = torch.randn(n, k, generator=gen).to(dtype)
    got, weight = moe.rms_norm_backward(x.cuda(), w.cuda(), g.cuda(), 1e-6, r.cuda())
    form = "whole" if k % (4 if dtype is F32 else 8) == 0 else "shifted"
    check(x, w, g, r, 1e-6, got, weight, dtype, form)
    before = torch.randn(k, generator=gen)
    got, weight = moe.rms_norm_backward(x.cuda(), w.cuda(), g.cuda(), 1e-6, r.cuda(), grad_weight=before.cuda())
    check(x, w, g, r, 1e-6, got, weight, dtype, form, before)
