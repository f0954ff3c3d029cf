"""GPU: the ways to the expert products on 8-bit banks beside the plain calls: with an estimate of the live assignments, with the library's own scratch, over a plan whose shared expert serves a part of
the tokens, and as the share of one rank under expert parallelism. Sums are exact, so whatever form a call takes, it has the bits of the plain call, which the 64-bit arithmetic checks elsewhere."""
import ctypes as C

import pytest
import torch

from test_gpu_int8 import experts_case, gen
from test_gpu_int8_guard import Guarded

pytestmark = pytest.mark.gpu


def device_banks(banks):
    from tqllm_b200 import moe
    return [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks] if banks else [None] * 3


def ref(b):
    return C.byref(b.c) if b is not None else None


@pytest.mark.parametrize("n,e,k,h,f,shared,route", ((1, 8, 2, 64, 48, False, "even"), (40, 16, 4, 256, 144, True, "skip"), (300, 6, 3, 144, 128, False, "skip"), (600, 3, 2, 2688, 208, True, "skip"),
                                                    (70, 4, 2, 128, 64, False, "none"), (260, 40, 2, 512, 256, False, "one")))
@pytest.mark.parametrize("family", ("auto", "gemm", "decode"))
def test_an_estimate_of_the_live_assignments(n, e, k, h, f, shared, route, family):
    """from none to all of them, right or not: the same bits, and rows of skipped assignments as they were"""
    from tqllm_b200 import capi, moe
    from tqllm_b200.capi import check, lib
    x, ids, banks, sh = experts_case(n, e, k, h, f, n + e, shared, route)
    dev, dsh, st = device_banks(banks), device_banks(sh), n if shared else 0
    xd, total = x.bfloat16().cuda(), n * k + st
    plan = moe.dispatch(ids.cuda(), e, st)
    full = lambda cols: torch.full((total, cols), 5.0, device="cuda")
    want = moe.expert_gateup_swiglu(dev[0], dev[1], xd, plan, dsh[0], dsh[1], act=full(f))
    rows = torch.randn(total, f, generator=gen(9)).cuda()
    want_y = moe.expert_down(dev[2], rows, plan, dsh[2], y=full(h))
    truth = int((ids >= 0).sum())
    with capi.family(family):
        for live in sorted({0, 1, truth, (truth + n * k) // 2, n * k}):
            act, y = full(f), full(h)
            size = lib.b2moe_expert_slot_workspace_bytes(ref(dev[0]), total, capi.BF16)
            ws = Guarded(max(size, lib.b2moe_expert_slot_workspace_bytes(ref(dev[2]), total, capi.F32)))
            check(lib.b2moe_expert_gateup_swiglu_sparse(ref(dev[0]), ref(dev[1]), ref(dsh[0]), ref(dsh[1]), xd.data_ptr(), capi.BF16, plan.buf.data_ptr(), n, k, st, live, act.data_ptr(), ws.ptr,
                                                        ws.size, moe._stream()), "gate/up")
            check(lib.b2moe_expert_down_sparse(ref(dev[2]), ref(dsh[2]), rows.data_ptr(), plan.buf.data_ptr(), n, k, st, live, y.data_ptr(), ws.ptr, ws.size, moe._stream()), "down")
            assert torch.equal(act, want) and torch.equal(y, want_y) and ws.intact(), live
        past = n * k + 1
        assert lib.b2moe_expert_down_sparse(ref(dev[2]), ref(dsh[2]), rows.data_ptr(), plan.buf.data_ptr(), n, k, st, past, y.data_ptr(), ws.ptr, ws.size, moe._stream()) == capi.ERR_SHAPE
    assert int(plan.buf[3]) == 0


def test_the_librarys_own_scratch():
    """calls of several sizes in turn: the array holds what the call before left"""
    from tqllm_b200 import capi, moe
    from tqllm_b200.capi import check, lib
    for n, e, k, h, f, shared, route in ((300, 8, 4, 256, 512, True, "skip"), (5, 8, 2, 64, 32, False, "even"), (40, 4, 2, 2688, 80, True, "even"), (300, 8, 4, 256, 512, False, "skip"), (3, 4, 2, 48, 16, True, "skip")):
        _, ids, banks, sh = experts_case(n, e, k, h, f, n, shared, route)
        down, shd, st = device_banks(banks)[2], device_banks(sh)[2], n if shared else 0
        plan = moe.dispatch(ids.cuda(), e, st)
        rows = torch.randn(n * k + st, f, generator=gen(2)).cuda()
        for family in ("auto", "gemm", "decode"):
            with capi.family(family):
                want, got = (torch.full((n * k + st, h), 5.0, device="cuda") for _ in range(2))
                moe.expert_down(down, rows, plan, shd, y=want)
                check(lib.b2moe_expert_down_static(ref(down), ref(shd), rows.data_ptr(), plan.buf.data_ptr(), n, k, st, got.data_ptr(), moe._stream()), "static")
                assert torch.equal(got, want)
        assert int(plan.buf[3]) == 0


@pytest.mark.parametrize("n,e,k,h,f,route", ((7, 4, 2, 64, 48, "even"), (200, 4, 2, 128, 144, "skip"), (300, 3, 2, 2688, 80, "even")))
@pytest.mark.parametrize("family", ("auto", "gemm", "decode"))
@pytest.mark.parametrize("room", ("rows", "slots"))
def test_a_shared_expert_for_a_part_of_the_tokens(n, e, k, h, f, route, family, room):
    """the rows of the range have the bits of a plan with all tokens, the shared rows of the others are left alone, nothing behind the buffers is written"""
    from tqllm_b200 import capi, moe
    from tqllm_b200.capi import check, lib
    x, ids, banks, sh = experts_case(n, e, k, h, f, 3, True, route)
    dev, dsh = device_banks(banks), device_banks(sh)
    xd, idd, total = x.half().cuda(), ids.cuda(), n * k + n
    every = moe.dispatch(idd, e, n)
    want = moe.expert_gateup_swiglu(dev[0], dev[1], xd, every, dsh[0], dsh[1], act=torch.full((total, f), 5.0, device="cuda"))
    rows = torch.randn(total, f, generator=gen(4)).cuda()
    want_y = moe.expert_down(dev[2], rows, every, dsh[2], y=torch.full((total, h), 5.0, device="cuda"))
    for first, count in ((0, n), (0, 1), (n - 1, 1), (n // 3, n // 2), (2, 0)):
        plan = moe.Plan(e, n, k, count, "cuda")
        dws = torch.empty(max(16, lib.b2moe_dispatch_workspace_bytes(e, n * k)), dtype=torch.uint8, device="cuda")
        check(lib.b2moe_dispatch_range(idd.data_ptr(), n, k, e, first, count, plan.buf.data_ptr(), dws.data_ptr(), dws.numel(), moe._stream()), "dispatch")
        up = lib.b2moe_expert_workspace_bytes(capi.I8, n, h, capi.F16) if room == "rows" else lib.b2moe_expert_slot_workspace_bytes(ref(dev[0]), total, capi.F16)
        down = lib.b2moe_expert_workspace_bytes(capi.I8, total, f, capi.F32) if room == "rows" else lib.b2moe_expert_slot_workspace_bytes(ref(dev[2]), total, capi.F32)
        ws_up, ws_down, act, y = Guarded(up), Guarded(down), Guarded(4 * total * f), Guarded(4 * total * h)
        act.floats(total, f).fill_(5.0)
        y.floats(total, h).fill_(5.0)
        with capi.family(family):
            check(lib.b2moe_expert_gateup_swiglu(ref(dev[0]), ref(dev[1]), ref(dsh[0]), ref(dsh[1]), xd.data_ptr(), capi.F16, plan.buf.data_ptr(), n, k, n, act.ptr, ws_up.ptr, up, moe._stream()), "up")
            check(lib.b2moe_expert_down(ref(dev[2]), ref(dsh[2]), rows.data_ptr(), plan.buf.data_ptr(), n, k, n, y.ptr, ws_down.ptr, down, moe._stream()), "down")
        served = torch.ones(total, dtype=torch.bool, device="cuda")
        served[n * k:] = False
        served[n * k + first:n * k + first + count] = True
        for got, exact in ((act.floats(total, f), want), (y.floats(total, h), want_y)):
            assert torch.equal(got[served], exact[served]) and bool((got[~served] == 5.0).all()), (first, count)
        assert all(b.intact() for b in (ws_up, ws_down, act, y)) and int(plan.buf[3]) == 0


def ranks_of(shape, router, banks, sh, world, vec):
    from tqllm_b200 import ep, moe
    e, out = router.shape[0], []
    for r in range(world):
        first, count = ep.expert_range(e, world, r)
        mine = [moe.DeviceBank.from_int8(w[first:first + count].cuda(), v[first:first + count].cuda()) for w, v in banks]
        layer = moe.MoeLayer.from_banks(shape, router[first:first + count], mine, device_banks(sh) if sh else None, shared_gate_vec=vec)
        out.append(ep.CudaEpLayer(layer, router, e, world, r, out_dtype=torch.float32))
    return out


@pytest.mark.parametrize("world,e,T", ((1, 8, 5), (2, 8, 3), (4, 24, 40), (3, 8, 200)))
@pytest.mark.parametrize("shared", ("none", "plain", "gated"))
@pytest.mark.parametrize("exchange", ("gather", "all-to-all"))
def test_a_ranks_share(world, e, T, shared, exchange):
    """All ranks on this device, the exchanges by copies. The rows are those of the unsplit layer to the bit; its output and the ranks' are 32-bit sums of the same k + 1 products in two orders:
    each is off by (k + 3) 2^-24 of the sum of their sizes at most (a product and k sums, the store of a part), so the two differ by twice that."""
    from tqllm_b200 import moe, synth
    k, h, f = (3 if exchange == "gather" else 4), 256, 144              # (records hold an even number of ids)
    x, _, banks, sh = experts_case(T * world, e, k, h, f, 8, shared != "none")
    shape = synth.LayerShape("i8-ranks", h, e, k, f, shared=shared != "none")
    router, vec = (torch.randn(e, h, generator=gen(1)) * 0.1).cuda(), (torch.randn(h, generator=gen(2)) * 0.1).cuda() if shared == "gated" else None
    xd = x.bfloat16().cuda()
    full = moe.MoeLayer.from_banks(shape, router, device_banks(banks), device_banks(sh) if sh else None, shared_gate_vec=vec)
    want = full.forward(xd)
    art = full.artefacts()
    y = art["y"].double()
    n = T * world
    size = (y[:n * k].view(n, k, h) * art["weights"].double()[..., None]).abs().sum(1)
    if sh:
        size += (y[n * k:] * (art["shared_weights"].double()[:, None] if vec is not None else 1.0)).abs()
    ranks = ranks_of(shape, router, banks, sh, world, vec)
    local = [xd[r * T:(r + 1) * T].contiguous() for r in range(world)]
    outs = []
    if exchange == "gather":
        routed = [rk.route_local(xl) for rk, xl in zip(ranks, local)]
        ids, w = torch.cat([i for i, _ in routed]), torch.cat([w for _, w in routed])
        assert torch.equal(ids, art["ids"])
        parts = [rk.partial_sums(xd, ids, w) for rk in ranks]
        for p, rk in enumerate(ranks):
            outs.append(rk.finish(torch.stack([parts[r][0][p * T:(p + 1) * T] for r in range(world)]).contiguous(), parts[p][1]).clone())
            assert int(rk.buf["plan"][3]) == 0
    else:
        st, backs = [], [[None] * world for _ in range(world)]
        for rk, xl in zip(ranks, local):
            ids, w = (t.clone() for t in rk.route_local(xl))
            counts, pos, lst = (t.clone() for t in rk.peer_lists(ids))
            m = counts.tolist()
            off = torch.tensor([sum(m[:i]) for i in range(world + 1)], dtype=torch.int32)
            st.append(dict(off=off.tolist(), offd=off.cuda(), pos=pos, send=rk.pack_records(xl, ids, w, lst, off.cuda(), sum(m)).clone(), sw=None if rk.shared_w is None else rk.shared_w.clone()))
        for p, rk in enumerate(ranks):
            segs = [s["send"][s["off"][p]:s["off"][p + 1]] for s in st]
            m = [s.shape[0] for s in segs]
            got, mine = rk.partial_sums_records(torch.cat(segs).contiguous(), sum(m), sum(m[:p]), T)
            assert int(rk.buf["plan"][3]) == 0
            st[p]["shared"] = None if mine is None else mine.clone()
            for r in range(world):
                backs[r][p] = got[sum(m[:r]):sum(m[:r + 1])].clone()
        for r, rk in enumerate(ranks):
            rk.shared_w = st[r]["sw"]
            outs.append(rk.finish_records(torch.cat(backs[r]).contiguous(), st[r]["pos"], st[r]["offd"], st[r]["shared"]).clone())
    got = torch.cat(outs).double()
    assert bool(((got - want.double()).abs() <= 2 * (k + 3) * 2.0 ** -24 * size + 1e-37).all())
