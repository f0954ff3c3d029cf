"""GPU: quantised rows, the dense 8-bit product and the expert products on 8-bit banks, against 64-bit arithmetic.

Bounds. Quantised rows and their scales are exact (64-bit floats decide every value). A product has an exact sum s and the
roundings of float(s), of the product of the scales, of their product and of the output type:
|y - exact| <= (3 * 2^-24 * (1 + 2^-20) + eps/2) |exact| + the smallest step of the type. act = g / (1 + exp(-g)) u: g and u carry
three roundings each, silu passes a relative error of g on times at most 1 + |g|, exp is off by 2 units in the last place, and there
are the roundings of the sum, the quotient and the product: (3 (1 + |g|) + 3 + 4 + 3) 2^-24, taken as (4 |g| + 16) 2^-24, and
exp(-g) overflows below -88, where |act| < 1e-35 |u|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def exact_rows(x):
    """(q, scale) of the definition; x on the CPU"""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(x).all(-1, keepdim=True)
    q = torch.round(127.0 * x / torch.where((top > 0) & fine, top, torch.ones_like(top)))
    q = torch.where(fine, q, torch.zeros_like(q))
    scale = torch.where(fine, (top.float() / 127.0).double(), torch.full_like(top, float("nan")))
    return q, scale[..., 0]


def exact_product(q, w):
    """whole numbers below 2^31: exact in 64-bit floats"""
    return q.double() @ w.double().T


def product_bound(exact, dtype):
    return (3 * 2.0 ** -24 * (1 + 2.0 ** -20) + torch.finfo(dtype).eps / 2) * exact.abs() + STEP[dtype]


def special_rows(k, dtype):
    """zeros, infinities, NaN, a single value, halves on both sides, the smallest and the largest values of the type"""
    f = torch.finfo(dtype)
    x = torch.zeros(9, k)
    x[1, 0] = float("inf")
    x[2, k - 1] = float("nan")
    x[3, k // 2] = -0.3
    x[4] = (torch.arange(k) % 255 - 127) * 0.5                         # top 63.5: whole numbers
    x[5] = (torch.arange(k) % 253 - 126) * 0.5
    x[5, 0] = 127.0                                                    # q = x: every other one a half
    x[6] = f.smallest_normal * (torch.arange(k) % 5 - 2) / 4
    x[7] = f.max * ((torch.arange(k) % 7) - 3) / 3
    x[8, 3] = f.tiny
    return x.to(dtype)


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("n,k", ((1, 16), (5, 48), (33, 512), (3, 528), (2, 4096), (7, 8208), (2, 16384), (3, 16400), (2, 131056)))
def test_quantized_rows(dtype, n, k):
    from tqllm_b200 import moe
    x = (torch.randn(n, k, generator=gen(n + k)) * torch.logspace(-3, 3, n)[:, None]).to(dtype)
    if k <= 4096:
        x = torch.cat([x, special_rows(k, dtype)])
    q, scale = moe.quantize_rows(x.cuda())
    want_q, want_scale = exact_rows(x)
    assert torch.equal(q.cpu().double(), want_q)
    assert torch.equal(torch.nan_to_num(scale.cpu().double(), nan=-1.0), torch.nan_to_num(want_scale, nan=-1.0))


def test_values_next_to_a_half():
    """fp32 neighbours of every half between two integers: the side is decided exactly"""
    from tqllm_b200 import moe
    rows = []
    for top in (1.0, 3.1415927, 0.7, 1.9999999, 1e-38, 1e-42, 3e38):
        t = torch.tensor(top, dtype=torch.float32)
        mid = ((torch.arange(-127, 127).double() + 0.5) * t.double() / 127.0).float()
        up, down = torch.nextafter(mid, torch.full_like(mid, 3.3e38)), torch.nextafter(mid, torch.full_like(mid, -3.3e38))
        rows.append(torch.cat([t[None], mid, up, down, torch.zeros(5)]))
    x = torch.stack(rows)
    q, _ = moe.quantize_rows(x.cuda())
    assert x.shape[1] == 768 and torch.equal(q.cpu().double(), exact_rows(x)[0])


def test_rows_of_a_wider_matrix():
    from tqllm_b200 import moe
    wide = torch.randn(6, 200, generator=gen(1)).bfloat16()
    q, scale = moe.quantize_rows(wide.cuda()[:, 8:104])
    want_q, want_scale = exact_rows(wide[:, 8:104])
    assert torch.equal(q.cpu().double(), want_q) and torch.equal(scale.cpu().double(), want_scale)


def linear_case(n, m, k, seed):
    g = gen(seed)
    q = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    return q, torch.rand(n, generator=g) * 0.1, w, torch.rand(m, generator=g) * 0.01


@pytest.mark.parametrize("n", (1, 2, 8, 9, 17, 33, 64, 100, 129, 300, 515))
@pytest.mark.parametrize("m,k", ((1, 16), (15, 48), (16, 64), (17, 80), (100, 1024), (257, 1040), (1411, 2560)))
@pytest.mark.parametrize("family", ("auto", "gemm", "decode"))
def test_linear(n, m, k, family):
    from tqllm_b200 import capi
    with capi.family(family):
        linear(n, m, k)


def linear(n, m, k):
    from tqllm_b200 import moe
    q, s, w, v = linear_case(n, m, k, n * 7 + m)
    bank = moe.DeviceBank.from_int8(w.cuda(), v.cuda())
    exact = exact_product(q, w) * s.double()[:, None] * v.double()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        y = moe.linear_i8(q.cuda(), s.cuda(), bank, out_dtype=dtype, status=status).cpu().double()
        assert bool(((y - exact).abs() <= product_bound(exact, dtype)).all()), dtype
    assert int(status) == 0


@pytest.mark.parametrize("n,m,k", ((1, 4096, 4096), (64, 4096, 4096), (200, 4096, 4096), (256, 130, 8192), (17, 70, 16400), (1000, 520, 4096), (2100, 1408, 1408), (700, 6500, 2688), (9000, 1300, 2688), (515, 4096, 4096), (1000, 1411, 2560)))
@pytest.mark.parametrize("family", ("auto", "gemm"))
def test_linear_of_real_sizes(n, m, k, family):
    from tqllm_b200 import capi
    with capi.family(family):
        linear_of_real_sizes(n, m, k)


def linear_of_real_sizes(n, m, k):
    from tqllm_b200 import moe
    q, s, w, v = linear_case(n, m, k, 3)
    y = moe.linear_i8(q.cuda(), s.cuda(), moe.DeviceBank.from_int8(w.cuda(), v.cuda()), out_dtype=torch.float32)
    exact = (q.cuda().double() @ w.cuda().double().T) * s.cuda().double()[:, None] * v.cuda().double()
    assert bool(((y.double() - exact).abs() <= product_bound(exact, torch.float32)).all())


@pytest.mark.parametrize("n", (1, 40, 200))
def test_the_largest_sums(n):
    """131,056 products of -128 and -128: 2^31 - 2^18"""
    from tqllm_b200 import moe
    k = (1 << 17) - 16
    q, w = torch.full((n, k), -128, dtype=torch.int8), torch.full((5, k), -128, dtype=torch.int8)
    w[1::2] = 127
    y = moe.linear_i8(q.cuda(), torch.ones(n).cuda(), moe.DeviceBank.from_int8(w.cuda(), torch.ones(5).cuda()), out_dtype=torch.float32).cpu()
    assert torch.equal(y[:, 0::2], torch.full((n, 3), float(16384 * k))) and torch.equal(y[:, 1::2], torch.full((n, 2), float(-128 * 127 * k)))


@pytest.mark.parametrize("n", (3, 70, 300))
def test_linear_on_rows_of_wider_matrices(n):
    from tqllm_b200 import moe
    q, s, w, v = linear_case(n, 77, 96, 5)
    wide = torch.randint(-128, 128, (n, 160), generator=gen(2), dtype=torch.int8)
    wide[:, 32:128] = q
    out = torch.full((n, 100), 7.0, dtype=torch.bfloat16, device="cuda")
    y = moe.linear_i8(wide.cuda()[:, 32:128], s.cuda(), moe.DeviceBank.from_int8(w.cuda(), v.cuda()), out=out[:, 11:88])
    exact = exact_product(q, w) * s.double()[:, None] * v.double()
    assert bool(((y.cpu().double() - exact).abs() <= product_bound(exact, torch.bfloat16)).all())
    assert bool((out[:, :11] == 7).all()) and bool((out[:, 88:] == 7).all())


def test_a_row_with_a_nan_stays_a_row():
    from tqllm_b200 import moe
    for n in (3, 150):
        x = torch.randn(n, 64, generator=gen(4))
        x[1, 5] = float("nan")
        x[2, 6] = float("-inf")
        q, s = moe.quantize_rows(x.cuda())
        w = torch.randn(50, 64, generator=gen(5)).cuda()
        y = moe.linear_i8(q, s, moe.DeviceBank.from_float(w), out_dtype=torch.float32)
        nan = torch.isnan(y).cpu()
        assert bool(nan[1:3].all()) and int(nan.sum()) == 100


def test_bank_of_floats_and_its_dump():
    from tqllm_b200 import moe
    w = torch.randn(3, 20, 48, generator=gen(6))
    bank = moe.DeviceBank.from_float(w.cuda())
    q, scale = exact_rows(w.view(60, 48))
    assert (bank.experts, bank.rows, bank.cols) == (3, 20, 48)
    assert torch.equal(bank.dequant().cpu(), q.float() * scale.float()[:, None])


# ---- expert products ----

def experts_case(n, e, k, h, f, seed, shared=False, route="even"):
    g = gen(seed)
    make = lambda x, r, c: (torch.randint(-127, 128, (x, r, c), generator=g, dtype=torch.int8), torch.rand(x, r, generator=g) * 0.02 / 127 + 1e-6)
    banks = [make(e, f, h), make(e, f, h), make(e, h, f)]
    sh = [make(1, f, h), make(1, f, h), make(1, h, f)] if shared else None
    ids = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(n)]).int()
    if route == "skip":
        ids[torch.rand(n, k, generator=g) < 0.5] = -1
        ids[0] = -1
    elif route == "one":
        ids[:] = -1
        ids[:, 0] = e - 1
    elif route == "none":
        ids[:] = -1
    elif route == "twice":                                             # the same expert in several slots of a token
        ids[:, 1:] = ids[:, :1]
    return torch.randn(n, h, generator=g), ids, banks, sh


def rows_of(ids, n, k, e, shared):
    """(assignment, token, expert) of every grouped assignment; expert e: the shared one"""
    flat = ids.flatten()
    a = [(i, i // k, int(flat[i])) for i in range(n * k) if flat[i] >= 0]
    return a + ([(n * k + t, t, e) for t in range(n)] if shared else [])


def pick(banks, sh, m, e, count):
    w, v = (banks if e < count else sh)[m]
    i = e if e < count else 0
    return w[i], v[i].double()


SHAPES = [  # n, e, k, h, f, shared, route
    (1, 8, 2, 64, 16, False, "even"), (3, 5, 5, 80, 48, True, "even"), (7, 16, 4, 256, 144, False, "skip"), (9, 4, 2, 48, 80, True, "skip"),
    (40, 3, 1, 128, 64, False, "one"), (17, 40, 6, 1040, 272, False, "even"), (130, 4, 2, 192, 208, True, "even"), (300, 6, 3, 144, 128, False, "skip"),
    (260, 2, 1, 128, 336, False, "one"), (5, 8, 2, 64, 32, False, "none"), (700, 8, 4, 512, 256, True, "even"), (1, 2, 1, 16, 16, False, "even"),
    (150, 4096, 2, 64, 32, False, "even"), (100, 4097, 2, 64, 32, True, "skip"), (5, 4, 4, 64, 48, True, "twice"), (70, 3, 3, 128, 144, False, "twice"), (60, 6, 2, 2576, 80, True, "even"), (600, 3, 2, 2688, 208, False, "skip"),
]


@pytest.mark.parametrize("n,e,k,h,f,shared,route", SHAPES)
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("room", ("rows", "slots"))
@pytest.mark.parametrize("family", ("auto", "gemm", "decode"))
def test_expert_products(n, e, k, h, f, shared, route, dtype, room, family):
    from tqllm_b200 import capi
    with capi.family(family):
        expert_products(n, e, k, h, f, shared, route, dtype, room)


def expert_products(n, e, k, h, f, shared, route, dtype, room):
    import ctypes as C

    from tqllm_b200 import capi, moe
    from tqllm_b200.capi import check, lib
    x, ids, banks, sh = experts_case(n, e, k, h, f, n + e, shared, route)
    x = x.to(dtype)
    dev = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks]
    dsh = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in sh] if shared else [None] * 3
    total, st = n * k + (n if shared else 0), n if shared else 0
    plan = moe.dispatch(ids.cuda(), e, st)
    ref = lambda b: C.byref(b.c) if b is not None else None
    act = torch.full((total, f), 5.0, device="cuda")
    size = (lib.b2moe_expert_workspace_bytes(capi.I8, n, h, moe._DT[dtype]) if room == "rows" else
            lib.b2moe_expert_slot_workspace_bytes(ref(dev[0]), total, moe._DT[dtype]))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    check(lib.b2moe_expert_gateup_swiglu(ref(dev[0]), ref(dev[1]), ref(dsh[0]), ref(dsh[1]), x.cuda().data_ptr(), moe._DT[dtype], plan.buf.data_ptr(), n, k, st, act.data_ptr(),
                                         ws.data_ptr(), size, moe._stream()), "gate/up")
    grouped = rows_of(ids, n, k, e, shared)
    q, s = exact_rows(x)
    got, seen = act.cpu().double(), torch.zeros(total, dtype=torch.bool)
    for x_id in sorted({g[2] for g in grouped}):
        rows = [(a, t) for a, t, i in grouped if i == x_id]
        at, tok = torch.tensor([r[0] for r in rows]), torch.tensor([r[1] for r in rows])
        seen[at] = True
        (wg, vg), (wu, vu) = pick(banks, sh, 0, x_id, e), pick(banks, sh, 1, x_id, e)
        gv, uv = exact_product(q[tok], wg) * s[tok][:, None] * vg, exact_product(q[tok], wu) * s[tok][:, None] * vu
        want = gv / (1 + torch.exp(-gv)) * uv
        bound = (4 * gv.abs() + 16) * 2.0 ** -24 * want.abs() + 1e-35 * uv.abs() + 2.0 ** -149
        assert bool(((got[at] - want).abs() <= bound).all()), x_id
    assert bool((got[~seen] == 5.0).all())                             # rows of skipped assignments stay as they were

    rows_in = torch.randn(total, f, generator=gen(9)) * 3
    rows_in[~seen] = float("nan")
    y = torch.full((total, h), 5.0, device="cuda")
    y = moe.expert_down(dev[2], rows_in.cuda(), plan, dsh[2], y=y).cpu().double()
    q, s = exact_rows(rows_in)
    for x_id in sorted({g[2] for g in grouped}):
        at = torch.tensor([a for a, _, i in grouped if i == x_id])
        w, v = pick(banks, sh, 2, x_id, e)
        want = exact_product(q[at], w) * s[at][:, None] * v
        assert bool(((y[at] - want).abs() <= product_bound(want, torch.float32)).all()), x_id
    assert bool((y[~seen] == 5.0).all())
    assert int(plan.buf[3]) == 0


@pytest.mark.parametrize("n", (1, 5, 64, 300))
@pytest.mark.parametrize("gating,shared", ((1, True), (2, False)))
def test_layer_on_8_bit_banks(n, gating, shared):
    """the layer call gives the bits of its parts called one by one, with a skip connection, and twice the same"""
    from tqllm_b200 import moe, synth
    e, k, h, f = 24, 3, 256, 144
    x, _, banks, sh = experts_case(n, e, k, h, f, 77, shared)
    shape = synth.LayerShape("i8", h, e, k, f, gating=gating, shared=shared)
    dev = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks]
    dsh = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in sh] if shared else None
    router = (torch.randn(e, h, generator=gen(1)) * 0.1).cuda()
    vec = (torch.randn(h, generator=gen(2)) * 0.1).cuda() if shared else None
    layer = moe.MoeLayer.from_banks(shape, router, dev, dsh, shared_gate_vec=vec)
    xd = x.bfloat16().cuda()
    out = layer.forward(xd)
    again = layer.forward(xd)
    res = torch.randn(n, h, generator=gen(3)).cuda()
    with_res = layer.forward(xd, residual=res)
    art = layer.artefacts()
    st = n if shared else 0
    plan = moe.dispatch(art["ids"].clone(), e, st)
    act = moe.expert_gateup_swiglu(dev[0], dev[1], xd, plan, *(dsh[:2] if shared else (None, None)))
    y = moe.expert_down(dev[2], act, plan, dsh[2] if shared else None)
    want = moe.combine(y, art["weights"], n, k, h, st, art["shared_weights"] if shared else None)
    assert torch.equal(out, want) and torch.equal(out, again) and art["status"] == 0
    assert bool(torch.isfinite(out).all()) and bool(((with_res - out - res).abs() <= 2.0 ** -22 * (out.abs() + res.abs()) + 1e-30).all())


@pytest.mark.parametrize("n", (3, 200))
def test_a_plan_with_a_shared_expert_and_a_call_without(n):
    """the shared expert's assignments are left alone"""
    from tqllm_b200 import capi, moe
    e, k, h, f = 4, 2, 128, 144
    x, ids, banks, _ = experts_case(n, e, k, h, f, 2, route="skip")
    dev = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks]
    shared, plain = moe.dispatch(ids.cuda(), e, n), moe.dispatch(ids.cuda(), e)
    for family in ("decode", "gemm"):
        with capi.family(family):
            want = moe.expert_gateup_swiglu(dev[0], dev[1], x.cuda(), plain)
            shared.shared_tokens = 0
            got = moe.expert_gateup_swiglu(dev[0], dev[1], x.cuda(), shared)
            assert torch.equal(got, want)
            assert torch.equal(moe.expert_down(dev[2], want, shared), moe.expert_down(dev[2], want, plain))


def test_per_matrix_calls():
    """the reference's call shapes on 8-bit banks: id lists and groups, 16-bit rows in and out"""
    import ctypes as C

    from tqllm_b200 import capi, moe
    from tqllm_b200.capi import check, lib
    for n, e, k, h, f in ((2, 6, 2, 64, 48), (50, 6, 2, 128, 80)):
        x, ids, banks, _ = experts_case(n, e, k, h, f, n)
        x = x.half()
        gate, up, down = (moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks)
        grouped = rows_of(ids, n, k, e, False)
        q, s = exact_rows(x)
        y = torch.empty(n * k, f, dtype=torch.bfloat16, device="cuda")
        size = lib.b2moe_expert_matvec_workspace_bytes(C.byref(gate.c), n, k)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        xd, idd = x.cuda(), ids.cuda()
        check(lib.b2moe_expert_matvec(C.byref(gate.c), xd.data_ptr(), capi.F16, y.data_ptr(), capi.BF16, idd.data_ptr(), n, k, 0, ws.data_ptr(), size, moe._stream()), "matvec")
        for a, t, i in grouped:
            want = exact_product(q[t:t + 1], banks[0][0][i]) * s[t] * banks[0][1][i].double()
            assert bool(((y[a].cpu().double() - want[0]).abs() <= product_bound(want[0], torch.bfloat16)).all())
        plan = moe.dispatch(idd, e)
        counts, groups = moe.plan_to_groups(plan)
        act = torch.empty(n * k, f, dtype=torch.float16, device="cuda")
        size = lib.b2moe_expert_gemm_gateup_workspace_bytes(C.byref(gate.c), n, k, capi.F16)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        check(lib.b2moe_expert_gemm_gateup(C.byref(gate.c), C.byref(up.c), xd.data_ptr(), capi.F16, act.data_ptr(), capi.F16, counts.data_ptr(), groups.data_ptr(), n, k,
                                           ws.data_ptr(), size, moe._stream()), "gate/up")
        want = moe.expert_gateup_swiglu(gate, up, xd, plan)
        assert torch.equal(act, want.half())
        size = lib.b2moe_expert_matvec_workspace_bytes(C.byref(down.c), n, k)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        out = torch.empty(n * k, h, dtype=torch.float16, device="cuda")
        check(lib.b2moe_expert_gemm(C.byref(down.c), act.data_ptr(), capi.F16, out.data_ptr(), capi.F16, counts.data_ptr(), groups.data_ptr(), n, k, 1, ws.data_ptr(), size,
                                    moe._stream()), "down")
        assert torch.equal(out, moe.expert_down(down, act.float(), plan).half())


@pytest.mark.parametrize("n,m,k", ((2, 130, 256), (200, 130, 256), (40, 300, 2560), (9000, 1300, 2688)))
def test_streams_and_graphs(n, m, k):
    """a call on another stream, and a captured decode step replayed with new tokens in the same buffers: every form of the product"""
    from tqllm_b200 import moe
    q, s, w, v = linear_case(n, m, k, 8)
    bank = moe.DeviceBank.from_int8(w.cuda(), v.cuda())
    x = torch.randn(n, k, generator=gen(1)).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = moe.linear_i8(*moe.quantize_rows(x), bank)
    stream.synchronize()
    assert torch.equal(side, moe.linear_i8(*moe.quantize_rows(x), bank))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = moe.linear_i8(*moe.quantize_rows(x), bank)
    for seed in (2, 3):
        x.copy_(torch.randn(n, k, generator=gen(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, moe.linear_i8(*moe.quantize_rows(x), bank))


def test_two_calls_at_once():
    """products on two streams whose blocks share the SMs and their tensor memory"""
    from tqllm_b200 import moe
    jobs = []
    for n, m, k in ((1000, 2000, 512), (9000, 1300, 2688), (40, 300, 2560), (3, 4096, 1024)):
        q, s, w, v = linear_case(n, m, k, n)
        bank = moe.DeviceBank.from_int8(w.cuda(), v.cuda())
        jobs.append((q.cuda(), s.cuda(), bank, moe.linear_i8(q.cuda(), s.cuda(), bank)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    outs = [[] for _ in jobs]
    for _ in range(20):
        for (q, s, bank, _), stream, out in zip(jobs, streams, outs):
            with torch.cuda.stream(stream):
                out.append(moe.linear_i8(q, s, bank))
    torch.cuda.synchronize()
    assert all(torch.equal(o, job[3]) for job, out in zip(jobs, outs) for o in out)


@pytest.mark.parametrize("n", (2, 90))
def test_a_captured_expert_block(n):
    """dispatch, gate/up, down and the weighted sum in one graph, replayed with other tokens and other ids"""
    from tqllm_b200 import moe
    e, k, h, f = 6, 3, 2688, 272
    _, _, banks, _ = experts_case(n, e, k, h, f, 5)
    dev = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks]
    x, ids, w = torch.zeros(n, h, device="cuda"), torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.rand(n, k, generator=gen(1)).cuda()

    def block():
        plan = moe.dispatch(ids, e)
        y = moe.expert_down(dev[2], moe.expert_gateup_swiglu(dev[0], dev[1], x, plan), plan)
        return moe.combine(y, w, n, k, h, ids=ids, out_dtype=torch.bfloat16)

    def fill(seed):
        a, b, _, _ = experts_case(n, e, k, h, f, seed, route="skip" if seed % 2 else "even")
        x.copy_(a)
        ids.copy_(b)

    fill(1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = block()
    for seed in (2, 3, 4):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, block())


@pytest.mark.parametrize("n", (3, 120))
@pytest.mark.parametrize("which", ("gate", "down"))
def test_a_layer_of_two_kinds_of_banks(n, which):
    """Q4_K experts on one side and 8-bit ones on the other: the layer call gives the bits of its parts"""
    from tqllm_b200 import moe, synth
    e, k, h, f = 16, 3, 256, 512
    shape = synth.LayerShape("mixed", h, e, k, f)
    raw = synth.make_layer(shape, 3, "cpu", experts=e)
    q4 = [moe.DeviceBank(synth.Q4_K, r.cuda(), e, *d) for r, d in zip(raw.raw, ((f, h), (f, h), (h, f)))]
    i8 = [moe.DeviceBank.from_float((torch.randn(e, *d, generator=gen(i)) * 0.02).cuda()) for i, d in enumerate(((f, h), (f, h), (h, f)))]
    banks = i8[:2] + q4[2:] if which == "gate" else q4[:2] + i8[2:]
    layer = moe.MoeLayer.from_banks(shape, raw.router_w.cuda(), banks)
    x = torch.randn(n, h, generator=gen(9)).bfloat16().cuda()
    out = layer.forward(x)
    art = layer.artefacts()
    assert art["status"] == 0 and torch.equal(out, layer.forward(x))
    # the parts: each side's product has the bits of a call of its own on what the layer handed it
    plan = moe.dispatch(art["ids"].clone(), e)
    if which == "gate":
        assert torch.equal(moe.expert_gateup_swiglu(*banks[:2], x, plan), art["act"])
    else:
        assert torch.equal(moe.expert_down(banks[2], art["act"].clone(), plan), art["y"])
    assert torch.equal(moe.combine(art["y"].clone(), art["weights"], n, k, h), out)


@pytest.mark.parametrize("n,m,k", ((40, 300, 2560), (300, 300, 256), (1500, 300, 2048), (9000, 1300, 2688)))
def test_a_wait_that_runs_out_is_reported(n, m, k):
    """one step's copies are left out (harness hook): the launch ends, sets the status word, and the next one is clean; the launches share columns in a cluster, walk
    alone and in pairs"""
    from tqllm_b200 import capi, moe
    q, s, w, v = linear_case(n, m, k, 6)
    bank, status = moe.DeviceBank.from_int8(w.cuda(), v.cuda()), torch.zeros(1, dtype=torch.int32, device="cuda")
    q, s = q.cuda(), s.cuda()
    clean = moe.linear_i8(q, s, bank, status=status)
    assert int(status) == 0
    capi.lib.b2moe_harness_wait_probe(1, 0)
    try:
        moe.linear_i8(q, s, bank, status=status)
        torch.cuda.synchronize()
    finally:
        capi.lib.b2moe_harness_wait_probe(-1, 0)
    assert int(status) != 0
    status.zero_()
    assert torch.equal(moe.linear_i8(q, s, bank, status=status), clean) and int(status) == 0


def test_a_wait_of_grouped_products_that_runs_out():
    from tqllm_b200 import capi, moe
    x, ids, banks, _ = experts_case(200, 4, 2, 256, 272, 3)
    dev = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks]
    plan = moe.dispatch(ids.cuda(), 4)
    xd = x.cuda()
    clean = moe.expert_gateup_swiglu(dev[0], dev[1], xd, plan)
    capi.lib.b2moe_harness_wait_probe(1, 0)
    try:
        moe.expert_gateup_swiglu(dev[0], dev[1], xd, plan)
        torch.cuda.synchronize()
    finally:
        capi.lib.b2moe_harness_wait_probe(-1, 0)
    assert int(plan.buf[3]) != 0
    plan = moe.dispatch(ids.cuda(), 4)
    assert torch.equal(moe.expert_gateup_swiglu(dev[0], dev[1], xd, plan), clean) and int(plan.buf[3]) == 0


def test_tensors_on_the_host_beside_those_on_the_device():
    from tqllm_b200 import capi, moe
    q, s, w, v = linear_case(4, 6, 32, 1)
    bank = moe.DeviceBank.from_int8(w.cuda(), v.cuda())
    l, ids = torch.zeros(5, 8).cuda(), torch.zeros(5, 2, dtype=torch.int32).cuda()
    b = moe.balance_loss(l, ids, 8, 0.1)
    calls = [lambda: moe.linear_i8(q.cuda(), s, bank), lambda: moe.linear_i8(q.cuda(), s.cuda(), moe.DeviceBank.from_int8(w, v)), lambda: moe.linear_i8(q.cuda(), s.cuda(), bank, out=torch.zeros(4, 6)),
             lambda: moe.balance_loss(l, ids.cpu(), 8, 0.1), lambda: moe.balance_loss(l, ids, 8, 0.1, mask=torch.ones(5, dtype=torch.bool)),
             lambda: moe.balance_loss(l, ids, 8, 0.1, offsets=torch.tensor([0, 5], dtype=torch.int32)), lambda: moe.balance_loss_backward(l, b, 2, 0.1, grad_loss=torch.tensor(1.0)),
             lambda: moe.balance_loss_backward(l, b, 2, 0.1, out=torch.zeros(5, 8))]
    for call in calls:
        with pytest.raises(capi.B2moeError) as e:
            call()
        assert e.value.status == capi.ERR_CUDA


@pytest.mark.parametrize("n,e,k,h,f,shared,route", [s for s in SHAPES if s[1] < 100])
def test_the_forms_give_the_same_bits(n, e, k, h, f, shared, route):
    from tqllm_b200 import capi, moe
    x, ids, banks, sh = experts_case(n, e, k, h, f, n * e, shared, route)
    dev = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in banks]
    dsh = [moe.DeviceBank.from_int8(w.cuda(), v.cuda()) for w, v in sh] if shared else [None] * 3
    plan = moe.dispatch(ids.cuda(), e, n if shared else 0)
    got = []
    for family in ("decode", "gemm"):
        with capi.family(family):
            act = moe.expert_gateup_swiglu(dev[0], dev[1], x.cuda(), plan, dsh[0], dsh[1])
            got.append((act, moe.expert_down(dev[2], act, plan, dsh[2]), moe.linear_i8(*moe.quantize_rows(x.cuda()), moe.DeviceBank.from_int8(dev[0].data[0], dev[0].aux[0]), out_dtype=torch.float32)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


# 16 warps (at most 296 blocks of 16 rows, 32 steps of 64 columns or more) and 8, with eight steps at once and the remainder behind them
@pytest.mark.parametrize("m,k", ((4736, 2048), (4737, 2048), (40, 2032), (40, 8192), (33, 9104), (4750, 4112), (9500, 2064), (7, 16400)))
@pytest.mark.parametrize("n", (1, 8, 9, 33))
def test_linear_streamed_by_few_and_many_warps(n, m, k):
    from tqllm_b200 import capi
    with capi.family("decode"):
        linear_of_real_sizes(n, m, k)
