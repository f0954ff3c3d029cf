"""GPU: calls whose kernels take tensor maps, as the first that a host thread makes (a serving thread that was handed pointers and a stream): nothing has bound the device's context to it yet."""
import ctypes as C
import threading

import pytest
import torch

from test_gpu_int8 import linear_case

pytestmark = pytest.mark.gpu


def in_a_new_thread(call):
    got = []
    thread = threading.Thread(target=lambda: got.append(call()))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    return got[0]


@pytest.mark.parametrize("n,m,k", ((40, 300, 2560), (300, 300, 256), (1500, 300, 2048)))
@pytest.mark.parametrize("captured", (False, True))
def test_dense_8_bit_product(n, m, k, captured):
    from tqllm_b200 import capi, moe
    q, s, w, v = (t.cuda() for t in linear_case(n, m, k, 6))
    bank, out = moe.DeviceBank.from_int8(w, v), torch.zeros(n, m, device="cuda")
    want = moe.linear_i8(q, s, bank, out_dtype=torch.float32)
    call = lambda stream: capi.lib.b2moe_linear_i8(q.data_ptr(), k, s.data_ptr(), C.byref(bank.c), n, out.data_ptr(), capi.F32, m, None, stream)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
            got = []
            thread = threading.Thread(target=lambda: got.append(call(stream.cuda_stream)))
            thread.start()
            thread.join()
        assert got == [capi.OK]
        graph.replay()
        torch.cuda.synchronize()
    else:
        assert in_a_new_thread(lambda: call(stream.cuda_stream)) == capi.OK
    assert torch.equal(out, want)


def test_router():
    from tqllm_b200 import capi, moe
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(512, 1024, generator=g).bfloat16().cuda(), (torch.randn(256, 1024, generator=g) * 0.1).cuda()
    want = moe.router(w, x)
    logits = torch.zeros_like(want)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    call = lambda: capi.lib.b2moe_router(w.data_ptr(), None, x.data_ptr(), capi.BF16, logits.data_ptr(), logits.stride(0), 1024, 256, 512, stream.cuda_stream)
    assert in_a_new_thread(call) == capi.OK
    assert torch.equal(logits, want)
