"""GPU: host threads that call the norm, the sorted rows, the gradients and the products with an epilogue at once, each on its own stream with sizes of its own: every call is served and has the bits that it has alone."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def case(seed, n, h, e, k, dtype):
    from tqllm_b200 import moe
    g = torch.Generator().manual_seed(seed)
    x, r = torch.randn(n, h, generator=g).to(dtype).cuda(), torch.randn(n, h, generator=g).to(dtype).cuda()
    w = torch.rand(h, generator=g).cuda()
    logits = torch.randn(n, e, generator=g).cuda()
    bank = moe.DeviceBank.from_float(torch.randn(300, h, generator=g).cuda())

    def step():
        norm = moe.rms_norm(x, w, 1e-6, r, quantize=True)
        ids, weights, _ = moe.topk_softmax(logits, e, k)
        plan = moe.dispatch(ids, e)
        rows, slots = moe.dispatch_rows(norm.y, ids, plan)
        out = moe.combine_rows(rows, slots, weights, n, k, residual=norm.sum)
        gy, gw, _ = moe.combine_rows_backward(out, rows, slots, weights, n, k)
        gl = moe.route_backward(logits, ids, weights, gw, e)
        gx = moe.dispatch_rows_backward(gy, slots, n, k)
        gh, dw = moe.rms_norm_backward(norm.sum, w, gx, 1e-6, out)
        return norm.y, norm.q, norm.scale, rows, slots, out, gw, gl, gh, dw, moe.linear_i8(norm.q, norm.scale, bank, activation="silu")
    return step


def test_at_once():
    steps = [case(*c) for c in ((1, 40, 256, 16, 4, torch.bfloat16), (2, 1300, 512, 64, 2, torch.float16), (3, 3, 4096, 8, 8, torch.float32), (4, 200, 2048, 32, 6, torch.bfloat16))]
    want = [s() for s in steps]
    torch.cuda.synchronize()
    bad, start = [], threading.Barrier(len(steps))

    def work(i):
        stream = torch.cuda.Stream()
        start.wait()
        with torch.cuda.stream(stream):
            for _ in range(40):
                got = steps[i]()
        stream.synchronize()
        if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
            bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
