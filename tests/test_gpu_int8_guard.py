"""GPU: what the expert products on 8-bit banks write stays inside the buffers they are given. Workspaces of exactly the documented sizes, `act` and `y` lie
inside larger ones whose bytes behind the end are known and have to be there after the call; with plans that hold a shared expert in calls that have none, too, whose assignments lie behind the routed ones."""
import ctypes as C

import pytest
import torch

from test_gpu_int8 import experts_case

pytestmark = pytest.mark.gpu
GUARD, BYTE = 1 << 20, 0xA5


class Guarded:
    """`size` bytes in front of a guard region"""

    def __init__(self, size: int):
        self.size, self.all = size, torch.full((size + GUARD,), BYTE, dtype=torch.uint8, device="cuda")

    @property
    def ptr(self):
        return self.all.data_ptr()

    def floats(self, *shape):
        return self.all[:self.size].view(torch.float32).view(*shape)

    def intact(self):
        return bool((self.all[self.size:] == BYTE).all())


@pytest.mark.parametrize("n,e,k,h,f", ((3, 4, 2, 128, 144), (200, 4, 2, 128, 144), (700, 6, 3, 144, 80), (300, 3, 3, 2688, 48)))
@pytest.mark.parametrize("route", ("even", "skip", "none"))
@pytest.mark.parametrize("family", ("decode", "gemm"))
@pytest.mark.parametrize("room", ("rows", "slots"))
@pytest.mark.parametrize("shared", ("neither", "plan", "both"))
def test_nothing_is_written_behind_the_buffers(n, e, k, h, f, route, family, room, shared):
    from tqllm_b200 import capi, moe
    from tqllm_b200.capi import check, lib
    x, ids, banks, sh = experts_case(n, e, k, h, f, 2, shared == "both", route)
    dev = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks]
    dsh = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in sh] if sh else [None] * 3
    ref = lambda b: C.byref(b.c) if b is not None else None
    st = n if shared == "both" else 0
    plan = moe.dispatch(ids.cuda(), e, 0 if shared == "neither" else n)
    total = n * k + st
    xd = x.bfloat16().cuda()
    if room == "rows":
        up, down = lib.b2moe_expert_workspace_bytes(capi.I8, n, h, capi.BF16), lib.b2moe_expert_workspace_bytes(capi.I8, total, f, capi.F32)
    else:
        up, down = lib.b2moe_expert_slot_workspace_bytes(ref(dev[0]), total, capi.BF16), lib.b2moe_expert_slot_workspace_bytes(ref(dev[2]), total, capi.F32)
    ws_up, ws_down, act, y = Guarded(up), Guarded(down), Guarded(4 * total * f), Guarded(4 * total * h)
    act.floats(total, f).fill_(0.0)
    with capi.family(family):
        check(lib.b2moe_expert_gateup_swiglu(ref(dev[0]), ref(dev[1]), ref(dsh[0]), ref(dsh[1]), xd.data_ptr(), capi.BF16, plan.buf.data_ptr(), n, k, st, act.ptr, ws_up.ptr, up,
                                             moe._stream()), "gate/up")
        check(lib.b2moe_expert_down(ref(dev[2]), ref(dsh[2]), act.ptr, plan.buf.data_ptr(), n, k, st, y.ptr, ws_down.ptr, down, moe._stream()), "down")
        want = None
        if shared == "plan":                                           # the same numbers as over a plan without the shared expert
            plain = moe.dispatch(ids.cuda(), e)
            want = moe.expert_gateup_swiglu(dev[0], dev[1], xd, plain)
    torch.cuda.synchronize()
    assert [b.intact() for b in (ws_up, ws_down, act, y)] == [True] * 4
    assert want is None or torch.equal(act.floats(total, f), want)
    assert int(plan.buf[3]) == 0
