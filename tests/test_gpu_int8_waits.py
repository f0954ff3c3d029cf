"""GPU: the tensor-core form of the 8-bit products when a wait runs out, at every place of a block's walk: the copies of its first step, of one whose place in the ring is used again, of the last two
(then the warp that issues the copies has ended before anyone misses them). The launch ends, says so, and the next one is right. The waits are cut short by leaving copies out (harness hook)."""
import contextlib

import pytest
import torch

from test_gpu_int8 import experts_case, linear_case

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def without_step(step):
    from tqllm_b200 import capi
    capi.lib.b2moe_harness_wait_probe(step, 0)
    try:
        yield
        torch.cuda.synchronize()
    finally:
        capi.lib.b2moe_harness_wait_probe(-1, 0)


# 21 steps of 128 columns an item: pairs of blocks with one item each, alone with two blocks an SM (two steps), clusters that share an item's columns (five steps a block)
DENSE = [(1536, 2048, 2688, s) for s in (0, 5, 19, 20)] + [(1500, 300, 256, s) for s in (0, 1)] + [(40, 300, 2560, s) for s in (0, 3)]


@pytest.mark.parametrize("n,m,k,step", DENSE)
def test_dense(n, m, k, step):
    from tqllm_b200 import moe
    q, s, w, v = linear_case(n, m, k, 6)
    bank, status = moe.DeviceBank.from_int8(w.cuda(), v.cuda()), torch.zeros(1, dtype=torch.int32, device="cuda")
    q, s = q.cuda(), s.cuda()
    clean = moe.linear_i8(q, s, bank, status=status)
    assert int(status) == 0
    with without_step(step):
        moe.linear_i8(q, s, bank, status=status)
    assert int(status) != 0
    status.zero_()
    assert torch.equal(moe.linear_i8(q, s, bank, status=status), clean) and int(status) == 0


@pytest.mark.parametrize("step", (0, 5, 20))
@pytest.mark.parametrize("which", ("gate/up", "down"))
def test_grouped_in_pairs(which, step):
    from tqllm_b200 import capi, moe
    n, e, k, h, f = 600, 2, 1, 2688, 2688
    x, ids, banks, _ = experts_case(n, e, k, h, f, 3)
    dev = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks]
    xd, idd = x.cuda(), ids.cuda()
    with capi.family("gemm"):
        call = (lambda p: moe.expert_gateup_swiglu(dev[0], dev[1], xd, p)) if which == "gate/up" else (lambda p: moe.expert_down(dev[2], xd, p))
        clean = call(moe.dispatch(idd, e))
        plan = moe.dispatch(idd, e)
        with without_step(step):
            call(plan)
        assert int(plan.buf[3]) != 0
        plan = moe.dispatch(idd, e)
        assert torch.equal(call(plan), clean) and int(plan.buf[3]) == 0
