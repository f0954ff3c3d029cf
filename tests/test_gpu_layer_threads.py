"""GPU: layer calls of two sizes from four host threads at once, each with its own workspace and stream: no thread's launch is refused for what another one's kernel takes of shared memory, and
every output has the bits of a call by itself."""
import ctypes as C

import pytest
import torch

from test_gpu_int8_threads import together

pytestmark = pytest.mark.gpu
Q4_K, IQ3_S, NVFP4G = 12, 21, 323


# two tokens route in one block, 40 in a cluster; decode kernels, the exact form and the grouped GEMM take more with longer rows or more experts
@pytest.mark.parametrize("types,layout,n", ((Q4_K, "codes", 2), (Q4_K, "codes", 40), (IQ3_S, "gguf", 8), (Q4_K, "codes", 120), (NVFP4G, "codes", 120)))
def test_layers(types, layout, n):
    from tqllm_b200 import capi, moe, synth
    from tqllm_b200.capi import lib
    calls, outs, want, keep = [], [], [], []
    for h, e, k, f in ((512, 8, 2, 256), (2048, 200, 2, 512)) * 2:
        shape = synth.LayerShape("threads", h, e, k, f, types=(types,) * 3)
        layer = moe.MoeLayer.from_synth(synth.make_layer(shape, 1, "cuda"), iq3s_layout=layout)
        x = torch.randn(n, h, generator=torch.Generator().manual_seed(h)).bfloat16().cuda()
        want.append(layer.forward(x).clone())
        out = torch.zeros(n, h, device="cuda")
        args = (C.byref(layer.c), x.data_ptr(), capi.BF16, n, out.data_ptr(), capi.F32, layer.ws.data_ptr(), layer.ws.numel())
        calls.append(lambda st, args=args: lib.b2moe_layer_forward(*args, st))
        keep.append((layer, x))
        outs.append(out)
    assert together(calls, 1500) == [0] * 4
    assert all(torch.equal(o, w) for o, w in zip(outs, want)) and all(layer.artefacts()["status"] == 0 for layer, _ in keep)
