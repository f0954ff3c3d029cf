"""GPU: host threads that call the 8-bit products at once, each on its own stream, with sizes that ask one kernel for different amounts of shared memory. A launch takes what its
call needs, whatever another thread's call has just asked for. The calls are those of the C ABI with arguments that are ready, which leave the threads side by side in the library most of the time."""
import ctypes as C
import sys
import threading

import pytest
import torch

from test_gpu_int8 import linear_case

pytestmark = pytest.mark.gpu


def together(calls, rounds):
    """calls: functions of a stream handle that return a status, a thread and a stream each; how many of the calls were refused"""
    refused, start = [0] * len(calls), threading.Barrier(len(calls))

    def work(i):
        stream, call, bad = torch.cuda.Stream(), calls[i], 0
        handle = stream.cuda_stream
        start.wait()
        for _ in range(rounds):
            bad += call(handle) != 0
        refused[i] = bad
        stream.synchronize()

    torch.cuda.synchronize()
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    return refused


# short and long rows (two blocks an SM and one), items of 128 and 192 rows of long ones; clusters with rings of nine and seven stages
@pytest.mark.parametrize("shapes", (((300, 300, 256), (1500, 1411, 2048)), ((40, 300, 2560), (200, 300, 2560))))
def test_dense(shapes):
    from tqllm_b200 import capi, moe
    from tqllm_b200.capi import lib
    calls, outs, want, keep = [], [], [], []
    for n, m, k in shapes * 2:
        q, s, w, v = (t.cuda() for t in linear_case(n, m, k, n))
        bank, out = moe.DeviceBank.from_int8(w, v), torch.zeros(n, m, device="cuda")
        args = (q.data_ptr(), k, s.data_ptr(), C.byref(bank.c), n, out.data_ptr(), capi.F32, m, None)
        calls.append(lambda st, args=args: lib.b2moe_linear_i8(*args, st))
        keep.append((q, s, bank))
        outs.append(out)
        want.append(moe.linear_i8(q, s, bank, out_dtype=torch.float32))
    assert together(calls, 5000) == [0] * len(calls)
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_grouped():
    from tqllm_b200 import capi, moe
    from tqllm_b200.capi import lib
    calls, outs, want, keep = [], [], [], []
    for n, e, k, h, f in ((64, 8, 2, 256, 128), (64, 600, 2, 2048, 128)) * 2:
        g = torch.Generator().manual_seed(e)
        gate, up = (moe.DeviceBank.from_int8(torch.randint(-127, 128, (e, f, h), generator=g, dtype=torch.int8).cuda(), torch.rand(e, f, generator=g).cuda() * 1e-3) for _ in range(2))
        x = torch.randn(n, h, generator=g).bfloat16().cuda()
        plan = moe.dispatch(torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(n)]).int().cuda(), e)
        size = lib.b2moe_expert_slot_workspace_bytes(C.byref(gate.c), n * k, capi.BF16)
        ws, act = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.zeros(n * k, f, device="cuda")
        args = (C.byref(gate.c), C.byref(up.c), None, None, x.data_ptr(), capi.BF16, plan.buf.data_ptr(), n, k, 0, act.data_ptr(), ws.data_ptr(), size)
        calls.append(lambda st, args=args: lib.b2moe_expert_gateup_swiglu(*args, st))
        keep.append((gate, up, x, plan, ws))
        outs.append(act)
        want.append((gate, up, x, plan))
    with capi.family("gemm"):
        want = [moe.expert_gateup_swiglu(*w) for w in want]
        assert together(calls, 3000) == [0] * len(calls)
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
