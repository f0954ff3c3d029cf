"""GPU: a launch of the 8-bit products that gives up a bounded wait shows it in its outputs, whether or not the caller brought a status word: what it did not finish is NaN. One step's copies of every
block are left out (harness hook), so that no item is finished. Everything beside the output stays as it was."""
import pytest
import torch

from test_gpu_int8 import experts_case, linear_case
from test_gpu_int8_waits import DENSE, without_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,m,k,step", DENSE)
@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
def test_dense(n, m, k, step, dtype):
    from tqllm_b200 import moe
    q, s, w, v = (t.cuda() for t in linear_case(n, m, k, 6))
    bank = moe.DeviceBank.from_int8(w, v)
    wide = torch.full((n + 2, m + 24), 7.0, dtype=dtype, device="cuda")
    out = wide[1:-1, 8:8 + m]
    with without_step(step):
        moe.linear_i8(q, s, bank, out=out)
    assert bool(torch.isnan(out).all())
    out.fill_(7.0)
    assert bool((wide == 7.0).all())
    moe.linear_i8(q, s, bank, out=out)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("n,h,f,step", ((600, 2688, 2688, 0), (600, 2688, 2688, 20), (200, 256, 272, 1)))
def test_grouped(n, h, f, step):
    from tqllm_b200 import capi, moe
    x, ids, banks, _ = experts_case(n, 2, 2, h, f, 3, route="skip")
    dev = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks]
    xd, live = x.cuda(), (ids.flatten() >= 0).cuda()
    plan = moe.dispatch(ids.cuda(), 2)
    act, y = torch.full((2 * n, f), 5.0, device="cuda"), torch.full((2 * n, h), 5.0, device="cuda")
    rows = torch.randn(2 * n, f, device="cuda")
    with capi.family("gemm"), without_step(step):
        moe.expert_gateup_swiglu(dev[0], dev[1], xd, plan, act=act)
        moe.expert_down(dev[2], rows, plan, y=y)
    for out in (act, y):
        assert bool(torch.isnan(out[live]).all()) and bool((out[~live] == 5.0).all())
