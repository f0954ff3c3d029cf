"""What stands before and behind the expert layer, forward and backward, as measurable cases: the norm, rows sorted by expert and brought
back with their weights, the gradient of the routing weights, and the 8-bit product with its epilogue.

A case is a dict of plain values:
  kind      "norm":       the skip connection is added and the sum normalised by its root mean square; out "y": rows of the input's type, "i8": rows of
                          8-bit integers with a scale each
            "norm_grad":  the norm's gradient on its rows (with the gradient that reaches them through the skip connection) and on its weight
            "rows":       tokens -> rows sorted by expert, and rows of expert outputs -> tokens, weighted, with shared expert and skip connection
            "rows_grad":  the gradients of both, on the expert outputs, the weights and the tokens
            "route_grad": the gradient of the routing weights on the logits; gating 1 softmax / 2 sigmoid
            "linear":     rows are normalised to 8 bits and multiplied with an 8-bit matrix [rows][cols]; bias, activation and skip connection follow
                          in the same pass
  dtype     type of the rows that come in and go out; weight_dtype: of the norm's weight
  skip      share of the assignments that another rank serves (id -1);  skew: the first expert gets about ten times the mean
  graph     the pass is captured once and replayed, as a decode loop does
"""
from __future__ import annotations

import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def _norm(name, tokens, cols, dtype, weight_dtype, out="y", residual=True, graph=False) -> dict:
    return dict(name=name, kind="norm", tokens=tokens, cols=cols, dtype=dtype, weight_dtype=weight_dtype, out=out, residual=residual, graph=graph)


def _norm_grad(name, tokens, cols, dtype, weight_dtype, residual=True, graph=False) -> dict:
    return dict(name=name, kind="norm_grad", tokens=tokens, cols=cols, dtype=dtype, weight_dtype=weight_dtype, residual=residual, graph=graph)


def _rows(name, kind, tokens, hidden, experts, topk, dtype, shared=False, skip=0.0, skew=False, graph=False) -> dict:
    return dict(name=name, kind=kind, tokens=tokens, hidden=hidden, experts=experts, topk=topk, dtype=dtype, shared=shared, skip=skip, skew=skew,
                graph=graph)


def _route_grad(name, tokens, experts, topk, gating=1, norm=True, scale=0.0, shared=False, graph=False) -> dict:
    return dict(name=name, kind="route_grad", tokens=tokens, experts=experts, topk=topk, gating=gating, norm=norm, scale=scale, shared=shared,
                graph=graph)


def _linear(name, tokens, cols, rows, dtype, activation="none", bias=True, residual=True, graph=False) -> dict:
    return dict(name=name, kind="linear", tokens=tokens, cols=cols, rows=rows, dtype=dtype, activation=activation, bias=bias, residual=residual,
                graph=graph)


def listed() -> list[dict]:
    return [
        # the norm in front of a decode step's 8-bit projections, a few users
        _norm("norm decode 8 to 8 bits", 8, 4096, "bf16", "f32", out="i8", graph=True),
        # the norm of a prefill chunk, with the running sum of the skip connections
        _norm("norm prefill 8192", 8192, 4096, "bf16", "bf16"),
        # a small model in fp32, an odd batch, whose norm is tuned
        _norm_grad("norm gradient 515 f32", 515, 2560, "f32", "f32"),
        # a training batch
        _norm_grad("norm gradient 8192", 8192, 4096, "bf16", "bf16"),
        # the decode step of 64 users on a layer of 512 small experts
        _rows("rows decode 64", "rows", 64, 2048, 512, 10, "bf16", shared=True, graph=True),
        # the prefill of a prompt on it
        _rows("rows prefill 4096", "rows", 4096, 2048, 512, 10, "bf16"),
        # a tuning batch on wide experts, half of the assignments on another rank
        _rows("rows gradient 509", "rows_grad", 509, 4096, 128, 8, "f16", skip=0.5),
        # a training batch on them whose load is skewed
        _rows("rows gradient 4093 skew", "rows_grad", 4093, 4096, 128, 8, "bf16", shared=True, skew=True),
        # a tuning step of a small router on a handful of tokens
        _route_grad("route gradient 48", 48, 32, 4, gating=2, scale=2.5, graph=True),
        # a training batch on 512 experts
        _route_grad("route gradient 8192", 8192, 512, 10, shared=True),
        # one token through a square projection in a decode loop
        _linear("linear decode 1", 1, 4096, 4096, "bf16", graph=True),
        # the prefill of a prompt through a projection with an activation
        _linear("linear prefill 4096", 4096, 4096, 4096, "bf16", activation="gelu"),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "norm_grad", "rows", "rows", "rows_grad", "rows_grad", "route_grad", "linear", "linear"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if kind in ("norm", "norm_grad"):
        weight_dtype = rng.choice([dtype, "f32"])
        cols = rng.choice([16 * _log_uniform(rng, 8, 1024), _log_uniform(rng, 100, 16384)])
        case = _norm("", _log_uniform(rng, 1, 8192), cols, dtype, weight_dtype) if kind == "norm" else _norm_grad("", _log_uniform(rng, 1, 8192), cols, dtype, weight_dtype)
        case["residual"] = rng.random() < 0.7
        if kind == "norm" and cols % 16 == 0 and rng.random() < 0.5:
            case["out"] = "i8"
    elif kind in ("rows", "rows_grad"):
        experts = _log_uniform(rng, 4, 512)
        topk = rng.randint(1, min(10, experts))
        case = _rows("", kind, _log_uniform(rng, 1, 8192), 8 * _log_uniform(rng, 32, 896), experts, topk, dtype)
        case["shared"] = rng.random() < 0.4
        case["skip"] = rng.choice([0.0, 0.0, 0.25, 0.75])
        case["skew"] = experts >= 32 and topk <= experts // 4 and rng.random() < 0.25
    elif kind == "route_grad":
        experts = _log_uniform(rng, 4, 1024)
        case = _route_grad("", _log_uniform(rng, 1, 8192), experts, rng.randint(1, min(10, experts)), rng.choice([1, 1, 2]))
        case["norm"] = case["gating"] == 1 or rng.random() < 0.6
        if case["norm"]:
            case["topk"] = max(2, case["topk"])                                         # one weight alone is always one
        case["scale"] = rng.choice([0.0, 1.0, 2.5])
        case["shared"] = case["gating"] == 1 and rng.random() < 0.5
    else:
        case = _linear("", _log_uniform(rng, 1, 8192), 16 * _log_uniform(rng, 8, 512), _log_uniform(rng, 64, 8192), dtype)
        case["activation"] = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])
        case["bias"], case["residual"] = rng.random() < 0.7, rng.random() < 0.7
    most = {k: max(work(c)[k] for c in listed() if c["kind"] == kind) for k in ("bytes", "flops")}
    while case["tokens"] > 1 and any(work(case)[k] > most[k] for k in most):
        case["tokens"] = max(1, case["tokens"] * 3 // 4)
    case["graph"] = case["tokens"] <= 64 and rng.random() < 0.5
    del case["name"]
    return case


def work(case) -> dict:
    n = case["tokens"]
    if case["kind"] in ("norm", "norm_grad"):
        k, e, r = case["cols"], SIZE[case["dtype"]], 1 if case["residual"] else 0
        weight = k * SIZE[case["weight_dtype"]]
        if case["kind"] == "norm":       # rows, skip connection, their sum, the normalised rows
            return {"bytes": float(n * k * (e + 2 * r * e) + weight + n * (k + 4 if case["out"] == "i8" else k * e)), "flops": 5.0 * n * k}
        return {"bytes": float(n * k * e * (3 + r) + weight + 4 * k), "flops": 9.0 * n * k}
    if case["kind"] in ("rows", "rows_grad"):
        h, e, k, s = case["hidden"], SIZE[case["dtype"]], case["topk"], 1 if case["shared"] else 0
        live = n * k * (1.0 - case["skip"]) + s * n
        if case["kind"] == "rows":       # tokens read, rows written, ids; rows read, skip connection read, tokens written, weights
            return {"bytes": n * h * e * 3.0 + 2.0 * live * h * e + n * (12.0 * k + 8.0 * s), "flops": 2.0 * live * h}
        # gradient of the tokens and rows read, gradients of rows and weights written; gradients of sorted rows read, of tokens written
        return {"bytes": n * h * e * 2.0 + 3.0 * live * h * e + n * (12.0 * k + 12.0 * s), "flops": 4.0 * live * h}
    if case["kind"] == "route_grad":
        k, cols = case["topk"], case["experts"] + (1 if case["shared"] else 0)
        return {"bytes": n * (12.0 * k + 4.0 * cols + (8.0 if case["shared"] else 0.0) + (4.0 * k if case["gating"] == 2 else 0.0)), "flops": 4.0 * n * k}
    k, m, e = case["cols"], case["rows"], SIZE[case["dtype"]]
    return {"bytes": float(n * k * e + 4 * k + m * (k + 4) + n * m * e * (2 if case["residual"] else 1) + (4 * m if case["bias"] else 0)), "flops": 2.0 * n * m * k}


def _popularity(case) -> list[float]:
    """probability that a token selects the expert"""
    e, k = case["experts"], case["topk"]
    if not case["skew"]:
        return [k / e] * e
    lo, hi = 0.0, 4.0
    for _ in range(40):
        a = 0.5 * (lo + hi)
        total = sum(r ** -a for r in range(1, e + 1))
        lo, hi = (a, hi) if e / total < 10.0 else (lo, a)
    return [min(1.0, k * r ** -a / total) for r in range(1, e + 1)]


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, n, k, dtype):
    """N(0, 1) with a few channels of large values, as the sums of skip connections have them"""
    x = _randn(g, n, k)
    x[:, :: max(1, k // 7)] *= 8.0
    return x.to(dtype)


class _State:
    """inputs of one case, and what a program that makes the call keeps"""


def _inputs(case, seed) -> _State:
    g, s, n = _gen(seed), _State(), case["tokens"]
    s.case, s.graph = case, None
    kind = case["kind"]
    if kind in ("norm", "norm_grad", "linear"):
        k, t = case["cols"], TORCH[case["dtype"]]
        s.x = _activations(g, n, k, t)
        s.weight = (_randn(g, k) * 0.1 + 1.0).to(TORCH[case.get("weight_dtype", "f32")])
    if kind == "norm":
        s.residual = (_randn(g, n, k) * 2.0).to(t) if case["residual"] else None
    elif kind == "norm_grad":
        s.grad = (_randn(g, n, k) * 1e-2).to(t)
        s.grad_sum = (_randn(g, n, k) * 1e-2).to(t) if case["residual"] else None
    elif kind in ("rows", "rows_grad"):
        h, e, k, t = case["hidden"], case["experts"], case["topk"], TORCH[case["dtype"]]
        keys = torch.rand(n, e, generator=g, device="cuda").log().neg()                 # exponential races: a sample without replacement
        s.ids = (keys / torch.tensor(_popularity(case), device="cuda")).topk(k, -1, largest=False).indices.to(torch.int32)
        if case["skip"]:
            s.ids[torch.rand(n, k, generator=g, device="cuda") < case["skip"]] = -1
        w = torch.rand(n, k, generator=g, device="cuda") + 0.1
        s.weights = w / w.sum(-1, keepdim=True)
        s.shared_weights = torch.rand(n, generator=g, device="cuda") if case["shared"] else None
        total = n * k + (n if case["shared"] else 0)
        s.y = (_randn(g, total, h) * 0.5).to(t)
        if kind == "rows":
            s.x = _activations(g, n, h, t)
            s.residual = (_randn(g, n, h) * 2.0).to(t)
            s.rows = torch.zeros(total, h, dtype=t, device="cuda")                      # rows behind the last assignment stay as they are
        else:
            s.slots = _sorted(s)[1]
            s.grad = (_randn(g, n, h) * 1e-2).to(t)
            s.grad_rows = (_randn(g, total, h) * 1e-2).to(t)
            s.grad_y = torch.zeros(total, h, dtype=t, device="cuda")
    elif kind == "route_grad":
        e, k = case["experts"], case["topk"]
        s.logits = _randn(g, n, e + (1 if case["shared"] else 0)) * 1.5
        p = torch.softmax(s.logits[:, :e], -1) if case["gating"] == 1 else torch.sigmoid(s.logits[:, :e])
        w, ids = p.topk(k, -1)
        if case["norm"]:
            w = w / w.sum(-1, keepdim=True)
        s.ids, s.weights = ids.to(torch.int32), (w * (case["scale"] or 1.0)).contiguous()
        s.grad = _randn(g, n, k) * 1e-2
        s.shared_weights = torch.sigmoid(s.logits[:, e]) if case["shared"] else None
        s.grad_shared = _randn(g, n) * 1e-2 if case["shared"] else None
    elif kind == "linear":
        w = _randn(g, case["rows"], k) * 0.02                                           # an 8-bit checkpoint: integers and a scale for each row
        top = w.abs().amax(-1)
        s.w, s.w_scale = torch.round(w * (127.0 / top)[:, None]).to(torch.int8), top / 127.0
        s.bias = _randn(g, case["rows"]) * 0.1 if case["bias"] else None
        s.residual = (_randn(g, n, case["rows"]) * 2.0).to(t) if case["residual"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] == "linear":
        from tqllm_b200 import moe
        s.bank = moe.DeviceBank.from_int8(s.w, s.w_scale)
    if case["graph"]:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _call(s)
        stream.synchronize()
        s.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s.graph, stream=stream):
            s.out = _call(s)
    return s


def run(state):
    if state.graph is not None:
        state.graph.replay()
        return state.out
    return _call(state)


def _call(s):
    return globals()[("_own_" if own else "_plain_") + s.case["kind"]](s)


# ---- the library's calls ----

def _own_norm(s):
    from tqllm_b200 import moe
    if s.case["out"] == "y":
        r = moe.rms_norm(s.x, s.weight, EPS, residual=s.residual)
        return {"y": r.y, "sum": r.sum} if s.residual is not None else r.y
    r = moe.rms_norm(s.x, s.weight, EPS, residual=s.residual, rows=False, quantize=True)
    y = r.q * r.scale[:, None]
    return {"y": y, "sum": r.sum} if s.residual is not None else y


def _own_norm_grad(s):
    from tqllm_b200 import moe
    grad, grad_weight = moe.rms_norm_backward(s.x, s.weight, s.grad, EPS, grad_sum=s.grad_sum)
    return {"x": grad, "weight": grad_weight}


def _own_rows(s):
    from tqllm_b200 import moe
    n, k = s.ids.shape
    plan = moe.dispatch(s.ids, s.case["experts"], n if s.case["shared"] else 0)
    rows, slots = moe.dispatch_rows(s.x, s.ids, plan, rows=s.rows)
    out = moe.combine_rows(s.y, slots, s.weights, n, k, shared_weights=s.shared_weights, residual=s.residual)
    return {"rows": rows, "slots": slots, "out": out}


def _own_rows_grad(s):
    from tqllm_b200 import moe
    n, k = s.ids.shape
    grad_y, grad_weights, grad_shared = moe.combine_rows_backward(s.grad, s.y, s.slots, s.weights, n, k, shared_weights=s.shared_weights, grad_y=s.grad_y)
    grad_x = moe.dispatch_rows_backward(s.grad_rows, s.slots, n, k)
    out = {"y": grad_y, "weights": grad_weights, "x": grad_x}
    return {**out, "shared": grad_shared} if s.case["shared"] else out


def _own_route_grad(s):
    from tqllm_b200 import moe
    c = s.case
    return moe.route_backward(s.logits, s.ids, s.weights, s.grad, c["experts"], gating=c["gating"], norm=c["norm"], scale=c["scale"],
                              shared_weights=s.shared_weights, grad_shared=s.grad_shared)


def _own_linear(s):
    from tqllm_b200 import moe
    r = moe.rms_norm(s.x, s.weight, EPS, rows=False, quantize=True)
    return moe.linear_i8(r.q, r.scale, s.bank, out_dtype=s.x.dtype, bias=s.bias, activation=s.case["activation"], residual=s.residual)


# ---- the plain forms ----

def _plain_quantized(h, w):
    """the norm's rows as integers and scales: the root mean square cancels in the integers; 64 bits decide the values next to a half"""
    u = h.double() * w.double()
    top = u.abs().amax(-1, keepdim=True)
    q = torch.round(u * 127.0 / top.clamp(min=1e-300)).float()
    return q, top.float() / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) / 127.0


def _plain_norm(s):
    t = s.x.dtype
    h = s.x.float() if s.residual is None else s.x.float() + s.residual.float()
    if s.case["out"] == "i8":
        q, scale = _plain_quantized(h, s.weight)
        y = q * scale
    else:
        y = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * s.weight.float()).to(t)
    return y if s.residual is None else {"y": y, "sum": h.to(t)}


def _plain_norm_grad(s):
    h, a = s.x.float(), s.grad.float() * s.weight.float()
    rho = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    grad = rho * (a - h * rho * rho * (a * h).mean(-1, keepdim=True))
    if s.grad_sum is not None:
        grad = grad + s.grad_sum.float()
    return {"x": grad.to(s.x.dtype), "weight": (s.grad.float() * h * rho).sum(0)}


def _sorted(s):
    """the assignments in expert order (those that are skipped behind the last) and the slot of every assignment; the shared expert's come last"""
    n, k = s.ids.shape
    e, total = s.case["experts"], s.y.shape[0]
    ids = s.ids.flatten().long()
    key = torch.where(ids < 0, e + 1, ids)
    if total > n * k:
        key = torch.cat([key, torch.full((n,), e, device="cuda")])
    order = torch.argsort(key, stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(total, device="cuda")
    return order, torch.where(key > e, -1, slots).to(torch.int32)


def _weighted(s, y, slots, weights, shared_weights):
    """rows of the slots back to their tokens, in 32 bits"""
    n, k = s.ids.shape
    at = slots.clamp(min=0).long()
    live = (slots >= 0).float()
    rows = y[at].float() * live[:, None]
    w = weights.flatten()
    out = (rows[: n * k] * w[:, None]).view(n, k, -1).sum(1)
    return out if shared_weights is None else out + rows[n * k :] * shared_weights[:, None]


def _plain_rows(s):
    n, k = s.ids.shape
    order, slots = _sorted(s)
    live = (slots >= 0)[order]
    token = torch.where(order < n * k, order // k, order - n * k)
    s.rows.copy_(torch.where(live[:, None], s.x[token], s.rows))
    out = _weighted(s, s.y, slots, s.weights, s.shared_weights) + s.residual.float()
    return {"rows": s.rows, "slots": slots, "out": out.to(s.y.dtype)}


def _plain_rows_grad(s):
    n, k = s.ids.shape
    at, live = s.slots.clamp(min=0).long(), s.slots >= 0
    token = torch.arange(n * k, device="cuda") // k
    w = s.weights.flatten()
    if s.case["shared"]:
        token, w = torch.cat([token, torch.arange(n, device="cuda")]), torch.cat([w, s.shared_weights])
    grad = s.grad.float()[token]
    grad_w = torch.where(live, (grad * s.y[at].float()).sum(-1), 0.0)
    padded = torch.cat([s.grad_y, s.grad_y[:1]])                                        # one row more, for the assignments that are skipped
    padded[torch.where(live, at, s.y.shape[0])] = (grad * w[:, None]).to(s.y.dtype)
    s.grad_y.copy_(padded[:-1])
    ones = torch.ones(n, device="cuda")
    grad_x = _weighted(s, s.grad_rows, s.slots, ones[:, None].expand(n, k), ones if s.case["shared"] else None)
    out = {"y": s.grad_y, "weights": grad_w[: n * k].view(n, k), "x": grad_x.to(s.y.dtype)}
    return {**out, "shared": grad_w[n * k :]} if s.case["shared"] else out


def _plain_route_grad(s):
    c, ids = s.case, s.ids.long()
    if c["norm"]:
        v = s.weights / (c["scale"] or 1.0)
        grad = s.weights * (v[:, None, :] * (s.grad[:, :, None] - s.grad[:, None, :])).sum(-1)
    else:
        grad = s.weights * s.grad
    if c["gating"] == 2:
        grad = grad / (1.0 + torch.exp(torch.gather(s.logits, 1, ids)))
    out = torch.zeros_like(s.logits).scatter_(1, ids, grad)
    if c["shared"]:
        out[:, c["experts"]] = s.grad_shared * s.shared_weights * (1.0 - s.shared_weights)
    return out


def _plain_linear(s):
    q, scale = _plain_quantized(s.x.float(), s.weight)
    y = (q @ s.w.float().T) * (scale * s.w_scale)
    if s.bias is not None:
        y = y + s.bias
    a = s.case["activation"]
    if a == "relu":
        y = y.clamp(min=0.0)
    elif a == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif a == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    elif a == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if s.residual is not None:
        y = y + s.residual.float()
    return y.to(s.x.dtype)


# ---- the definitions in 64 bits ----

def exact(case, seed):
    return globals()["_exact_" + case["kind"]](_inputs(case, seed), case)


def _root(h):
    return h.square().mean(-1, keepdim=True).add(EPS).sqrt()


def _integers(h, w):
    """(the integers, the scales) of the norm's rows: the integers nearest to 127 u / max|u| for u = h w, products that 64 bits hold exactly"""
    u = h * w
    top = u.abs().max(-1, keepdim=True).values
    return torch.round(127.0 * u / torch.where(top > 0, top, torch.ones_like(top))), top / _root(h) / 127.0


def _exact_norm(s, case):
    # the sum is a 32-bit number; everything behind it starts from there
    h = (s.x.float() if s.residual is None else s.x.float() + s.residual.float()).double()
    if case["out"] == "i8":
        q, scale = _integers(h, s.weight.double())
        y = q * scale
    else:
        y = h / _root(h) * s.weight.double()
    return y if s.residual is None else {"y": y, "sum": h}


def _exact_norm_grad(s, case):
    h = s.x.double().requires_grad_()
    w = s.weight.double().requires_grad_()
    with torch.enable_grad():
        y = h / _root(h) * w
        gx, gw = torch.autograd.grad(y, (h, w), s.grad.double())
    return {"x": gx if s.grad_sum is None else gx + s.grad_sum.double(), "weight": gw}


def _exact_rows(s, case):
    n, k = s.ids.shape
    rows, slots, first = torch.zeros_like(s.rows), torch.full((s.y.shape[0],), -1, dtype=torch.int32, device="cuda"), 0
    for e in range(case["experts"]):
        a = (s.ids.flatten() == e).nonzero()[:, 0]
        rows[first : first + a.numel()] = s.x[a // k]
        slots[a] = torch.arange(first, first + a.numel(), device="cuda", dtype=torch.int32)
        first += a.numel()
    out = s.residual.double()
    if case["shared"]:
        rows[first : first + n] = s.x
        slots[n * k :] = torch.arange(first, first + n, device="cuda", dtype=torch.int32)
        out = out + s.shared_weights.double()[:, None] * s.y[first : first + n].double()
    for j in range(k):
        t = (slots[: n * k].view(n, k)[:, j] >= 0).nonzero()[:, 0]
        out[t] += s.weights[t, j].double()[:, None] * s.y[slots[t * k + j].long()].double()
    return {"rows": rows.double(), "slots": slots, "out": out}


def _exact_rows_grad(s, case):
    n, k = s.ids.shape
    grad = s.grad.double()
    gy, gw, gx = torch.zeros_like(s.y, dtype=torch.float64), torch.zeros(n, k, dtype=torch.float64, device="cuda"), torch.zeros_like(grad)
    for j in range(k):
        t = (s.slots[: n * k].view(n, k)[:, j] >= 0).nonzero()[:, 0]
        at = s.slots[t * k + j].long()
        gy[at] = s.weights[t, j].double()[:, None] * grad[t]
        gw[t, j] = torch.einsum("th,th->t", grad[t], s.y[at].double())
        gx[t] += s.grad_rows[at].double()
    out = {"y": gy, "weights": gw, "x": gx}
    if case["shared"]:
        at = s.slots[n * k :].long()
        gy[at] = s.shared_weights.double()[:, None] * grad
        out["shared"] = torch.einsum("th,th->t", grad, s.y[at].double())
        gx += s.grad_rows[at].double()
    return out


def _exact_route_grad(s, case):
    w, g, l, e = s.weights.double(), s.grad.double(), s.logits.double(), case["experts"]
    out = torch.zeros_like(l)
    if case["norm"]:
        share = w / (case["scale"] or 1.0)
        each = sum(share[:, i : i + 1] * (g - g[:, i : i + 1]) for i in range(case["topk"])) * w
    else:
        each = w * g
    for j in range(case["topk"]):
        at = s.ids[:, j : j + 1].long()
        d = each[:, j : j + 1]
        out.scatter_(1, at, d * torch.sigmoid(-l.gather(1, at)) if case["gating"] == 2 else d)
    if case["shared"]:
        p = s.shared_weights.double()
        out[:, e] = s.grad_shared.double() * p * (1.0 - p)
    return out


def _exact_linear(s, case):
    q, scale = _integers(s.x.double(), s.weight.double())
    y = (q @ s.w.double().T) * scale * s.w_scale.double()
    if case["bias"]:
        y = y + s.bias.double()
    f = torch.nn.functional
    y = {"none": lambda v: v, "relu": f.relu, "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh")}[case["activation"]](y)
    return y + s.residual.double() if case["residual"] else y
