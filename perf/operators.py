"""Operators beside the quantised-block path, as measurable cases: products of 8-bit integers with a scale for each token and
each channel (dense, and grouped by expert), and the router's balance loss with its gradient.

A case is a dict of plain values:
  kind      "linear":  rows x [tokens][cols] are quantised to 8 bits and multiplied with an 8-bit matrix [rows][cols]
            "experts": the expert block of a MoE layer on 8-bit banks, from ids and weights to the combined rows: dispatch, gate/up
                       + SwiGLU, down, weighted sum
            "balance": the balance loss of a batch of routed tokens, with the counts per expert, and its gradient
  dtype     type of the rows that come in and go out
  skip      "experts": share of the assignments that another rank serves (id -1)
  skew      "experts": the first expert gets about ten times the mean
  sequences, mask, gating   "balance": sequences of ragged length, padded tokens among them, 1 softmax / 2 normalised sigmoid
  graph     the pass is captured once and replayed, as a decode loop does
"""
from __future__ import annotations

import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _linear(name, tokens, cols, rows, dtype, graph=False) -> dict:
    return dict(name=name, kind="linear", tokens=tokens, cols=cols, rows=rows, dtype=dtype, graph=graph)


def _experts(name, tokens, hidden, experts, topk, ff, dtype, skip=0.0, skew=False, graph=False) -> dict:
    return dict(name=name, kind="experts", tokens=tokens, hidden=hidden, experts=experts, topk=topk, ff=ff, dtype=dtype, skip=skip, skew=skew,
                graph=graph)


def _balance(name, tokens, experts, topk, gating=1, sequences=1, mask=False, graph=False) -> dict:
    return dict(name=name, kind="balance", tokens=tokens, experts=experts, topk=topk, gating=gating, sequences=sequences, mask=mask, graph=graph)


def listed() -> list[dict]:
    return [
        # one token through a square projection in a decode loop: launches and weight streaming
        _linear("linear decode 1", 1, 4096, 4096, "bf16", graph=True),
        # a batch of drafts through a ragged output head
        _linear("linear 77 ragged", 77, 2560, 1411, "f16"),
        # a small model in fp32, an odd chunk
        _linear("linear 515 f32", 515, 1408, 4096, "f32"),
        # the prefill of long prompts through a square projection
        _linear("linear prefill 8192", 8192, 4096, 4096, "bf16"),
        # one chat user on a layer of 512 small experts
        _experts("experts decode 1", 1, 2048, 512, 10, 512, "bf16", graph=True),
        # the decode step of 64 users on it: nearly every expert is read for one or two tokens
        _experts("experts decode 64", 64, 2048, 512, 10, 512, "bf16", graph=True),
        # a chunk of a prefill on wide experts, half of the assignments on another rank
        _experts("experts chunk 509", 509, 4096, 128, 8, 1408, "f16", skip=0.5),
        # the prefill of a prompt on the layer of small experts
        _experts("experts prefill 4096", 4096, 2048, 512, 10, 512, "bf16"),
        # the same on wide experts whose load is skewed
        _experts("experts prefill 2047 skew", 2047, 4096, 128, 8, 1408, "bf16", skew=True),
        # a tuning step of a small router on a handful of tokens
        _balance("balance 48", 48, 32, 4, graph=True),
        # a training batch on 512 experts
        _balance("balance 8192", 8192, 512, 10),
        # the loss sequence by sequence over a padded batch, sigmoid scores
        _balance("balance sequences 6001", 6001, 128, 8, gating=2, sequences=12, mask=True),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng) -> dict:
    kind = rng.choice(["linear", "linear", "experts", "experts", "balance"])
    if kind == "linear":
        case = _linear("", _log_uniform(rng, 1, 8192), 16 * _log_uniform(rng, 8, 512), _log_uniform(rng, 64, 8192), rng.choice(["bf16", "f16", "f32"]))
        case["graph"] = case["tokens"] <= 64 and rng.random() < 0.5
    elif kind == "experts":
        experts = _log_uniform(rng, 4, 512)
        hidden, ff = 16 * _log_uniform(rng, 16, 256), 16 * _log_uniform(rng, 8, 96)
        while 3 * experts * hidden * ff > 2.3e9:
            experts //= 2
        topk = rng.randint(1, min(10, experts))
        case = _experts("", _log_uniform(rng, 1, 4096), hidden, experts, topk, ff, rng.choice(["bf16", "f16"]))
        case["skip"] = rng.choice([0.0, 0.0, 0.25, 0.75])
        case["skew"] = experts >= 32 and topk <= experts // 4 and rng.random() < 0.25
        case["graph"] = case["tokens"] <= 64 and rng.random() < 0.5
    else:
        experts = _log_uniform(rng, 4, 1024)
        tokens = _log_uniform(rng, 1, 8192)
        case = _balance("", tokens, experts, rng.randint(1, min(10, experts)), rng.choice([1, 1, 2]))
        case["sequences"] = rng.choice([1, _log_uniform(rng, 1, min(64, tokens))])
        case["mask"] = rng.random() < 0.4
        case["graph"] = tokens <= 64 and rng.random() < 0.5
    most = {k: max(work(c)[k] for c in listed() if c["kind"] == kind) for k in ("bytes", "flops")}
    while case["tokens"] > 1 and any(work(case)[k] > most[k] for k in most):
        case["tokens"] = max(1, case["tokens"] * 3 // 4)
    if kind == "balance":
        case["sequences"] = min(case["sequences"], case["tokens"])
    del case["name"]
    return case


def work(case) -> dict:
    n = case["tokens"]
    if case["kind"] == "linear":
        k, m, e = case["cols"], case["rows"], SIZE[case["dtype"]]
        return {"bytes": float(n * k * e + m * (k + 4) + n * m * e), "flops": 2.0 * n * m * k}
    if case["kind"] == "experts":
        # ids, weights and rows once, the banks of the experts that are expected to be touched, the combined rows
        h, f, experts, e = case["hidden"], case["ff"], case["experts"], SIZE[case["dtype"]]
        live = n * case["topk"] * (1.0 - case["skip"])
        touched = sum(1.0 - (1.0 - min(1.0, p * (1.0 - case["skip"]))) ** n for p in _popularity(case))
        return {"bytes": touched * (3.0 * h * f + 4.0 * (2 * f + h)) + n * (2.0 * h * e + 8.0 * case["topk"]), "flops": 6.0 * live * h * f}
    # logits read for the loss and again for the gradient, ids, mask; the gradient, counts and mean probabilities written
    experts = case["experts"]
    return {"bytes": 12.0 * n * experts + 4.0 * n * case["topk"] + (n if case["mask"] else 0) + 8.0 * case["sequences"] * experts, "flops": 12.0 * n * experts}


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


def _matrix(g, *shape):
    """an 8-bit checkpoint of N(0, 0.02) weights: integers and a scale for each row"""
    w = torch.randn(*shape, generator=g, device="cuda") * 0.02
    top = w.abs().amax(-1)
    return torch.round(w * (127.0 / top)[..., None]).to(torch.int8), top / 127.0


def _rows(g, n, k, dtype):
    """activations: N(0, 1) with a few channels of large values, as the inputs of such layers have them"""
    x = torch.randn(n, k, generator=g, device="cuda")
    x[:, :: max(1, k // 7)] *= 8.0
    return x.to(dtype)


def _top(g, case):
    """routed ids (distinct in a token) and weights that add up to one"""
    keys = torch.rand(case["tokens"], case["experts"], generator=g, device="cuda").log().neg()      # exponential races: a sample without replacement
    p = torch.tensor(_popularity(case) if "skew" in case else [1.0] * case["experts"], device="cuda")
    ids = (keys / p).topk(case["topk"], -1, largest=False).indices.to(torch.int32)
    w = torch.rand(case["tokens"], case["topk"], generator=g, device="cuda") + 0.1
    return ids, w / w.sum(-1, keepdim=True)


class _State:
    """inputs of one case, and what a program that makes the call keeps"""


def _inputs(case, seed) -> _State:
    g, s, n = _gen(seed), _State(), case["tokens"]
    s.case, s.pool, s.graph = case, None, None
    if case["kind"] == "linear":
        s.x = _rows(g, n, case["cols"], TORCH[case["dtype"]])
        s.w, s.w_scale = _matrix(g, case["rows"], case["cols"])
    elif case["kind"] == "experts":
        e, h, f = case["experts"], case["hidden"], case["ff"]
        s.x = _rows(g, n, h, TORCH[case["dtype"]])
        s.ids, s.weights = _top(g, case)
        if case["skip"]:
            s.ids[torch.rand(n, case["topk"], generator=g, device="cuda") < case["skip"]] = -1
        s.gate, s.gate_scale = _matrix(g, e, f, h)
        s.up, s.up_scale = _matrix(g, e, f, h)
        s.down, s.down_scale = _matrix(g, e, h, f)
        s.room = max(1, int(torch.bincount(s.ids.flatten().long() + 1, minlength=e + 1)[1:].max()))       # tokens of the fullest expert
    else:
        e = case["experts"]
        s.logits = torch.randn(n, e, generator=g, device="cuda") * 1.5 + torch.randn(e, generator=g, device="cuda") * 0.5
        s.ids = s.logits.topk(case["topk"], -1).indices.to(torch.int32)
        cuts = torch.randperm(max(n - 1, 1), generator=g, device="cuda")[: case["sequences"] - 1].sort().values + 1
        ends = torch.tensor([0], device="cuda"), cuts, torch.tensor([n], device="cuda")
        s.offsets = torch.cat(ends).to(torch.int32)
        s.mask = (torch.rand(n, generator=g, device="cuda") < 0.8) if case["mask"] else None
        s.coef = 0.01
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _handles(s)
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
    if own:
        return {"linear": _own_linear, "experts": _own_experts, "balance": _own_balance}[s.case["kind"]](s)
    return {"linear": _plain_linear, "experts": _plain_experts, "balance": _plain_balance}[s.case["kind"]](s)


# ---- the library's calls ----

def _handles(s):
    """banks over the checkpoint's arrays, as a loaded model holds them"""
    from tqllm_b200 import moe
    if s.case["kind"] == "linear":
        s.bank = moe.DeviceBank.from_int8(s.w, s.w_scale)
    elif s.case["kind"] == "experts":
        s.banks = [moe.DeviceBank.from_int8(w, v) for w, v in ((s.gate, s.gate_scale), (s.up, s.up_scale), (s.down, s.down_scale))]


def _own_linear(s):
    from tqllm_b200 import moe
    q, scale = moe.quantize_rows(s.x)
    return moe.linear_i8(q, scale, s.bank, out_dtype=s.x.dtype)


def _own_experts(s):
    from tqllm_b200 import moe
    n, k = s.ids.shape
    gate, up, down = s.banks
    plan = moe.dispatch(s.ids, s.case["experts"])
    act = moe.expert_gateup_swiglu(gate, up, s.x, plan, act=torch.empty(n * k, gate.rows, device="cuda"))
    y = moe.expert_down(down, act, plan, y=torch.empty(n * k, down.rows, device="cuda"))
    return moe.combine(y, s.weights, n, k, down.rows, ids=s.ids, out_dtype=s.x.dtype)


def _own_balance(s):
    from tqllm_b200 import moe
    c = s.case
    b = moe.balance_loss(s.logits, s.ids, c["experts"], s.coef, gating=c["gating"], mask=s.mask, offsets=s.offsets)
    grad = moe.balance_loss_backward(s.logits, b, c["topk"], s.coef, gating=c["gating"], mask=s.mask, offsets=s.offsets)
    return {"loss": b.loss, "counts": b.counts, "prob": b.prob, "grad": grad}


# ---- the plain forms ----

def _plain_quantize(x):
    """the nearest integers to 127 x / max|x|: 64 bits decide the values next to a half"""
    top = x.float().abs().amax(-1, keepdim=True)
    q = torch.round(x.double() * 127.0 / top.double().clamp(min=1e-300))
    return q.float(), top / 127.0


def _plain_linear(s):
    q, scale = _plain_quantize(s.x)
    return ((q @ s.w.float().T) * (scale * s.w_scale)).to(s.x.dtype)


def _plain_experts(s):
    """rows sorted into a block of each expert; where the assignments are fewer than the experts, the matrices of each assignment instead"""
    n, k = s.ids.shape
    e, room = s.case["experts"], s.room
    if n * k < e:
        at = s.ids.flatten().clamp(min=0).long()
        q, scale = (v.repeat_interleave(k, 0)[:, None] for v in _plain_quantize(s.x))
        g = (q @ s.gate[at].float().transpose(1, 2)) * (scale * s.gate_scale[at][:, None])
        u = (q @ s.up[at].float().transpose(1, 2)) * (scale * s.up_scale[at][:, None])
        q2, scale2 = _plain_quantize(g / (1.0 + torch.exp(-g)) * u)
        y = (q2 @ s.down[at].float().transpose(1, 2)) * (scale2 * s.down_scale[at][:, None])
        return (y.view(n, k, -1) * torch.where(s.ids < 0, 0.0, s.weights)[..., None]).sum(1).to(s.x.dtype)
    ids = s.ids.flatten().long()
    order = torch.argsort(torch.where(ids < 0, e, ids), stable=True)
    sorted_ids = torch.where(ids < 0, e, ids)[order]
    counts = torch.zeros(e + 1, dtype=torch.long, device="cuda").scatter_add_(0, sorted_ids, torch.ones_like(sorted_ids))
    place = torch.arange(n * k, device="cuda") - (counts.cumsum(0) - counts)[sorted_ids]
    place = torch.where(sorted_ids < e, sorted_ids * room + place, e * room)            # skipped assignments: one row behind the last
    slot = torch.empty_like(place)
    slot[order] = place
    q, scale = _plain_quantize(s.x)
    rows = torch.zeros(e * room + 1, q.shape[1], device="cuda")
    rows[place] = q[order // k]
    rows_scale = torch.zeros(e * room + 1, 1, device="cuda")
    rows_scale[place] = scale[order // k]
    b, bs = rows[:-1].view(e, room, -1), rows_scale[:-1].view(e, room, 1)
    g = (b @ s.gate.float().transpose(1, 2)) * (bs * s.gate_scale[:, None])
    u = (b @ s.up.float().transpose(1, 2)) * (bs * s.up_scale[:, None])
    q2, scale2 = _plain_quantize(g / (1.0 + torch.exp(-g)) * u)
    y = (q2 @ s.down.float().transpose(1, 2)) * (scale2 * s.down_scale[:, None])
    y = torch.cat([y.reshape(e * room, -1), torch.zeros(1, y.shape[2], device="cuda")])
    return (y[slot].view(n, k, -1) * s.weights[..., None]).sum(1).to(s.x.dtype)


def _plain_balance(s):
    c = s.case
    e, k, q, n = c["experts"], c["topk"], c["sequences"], c["tokens"]
    of = (torch.arange(n, device="cuda")[:, None] >= s.offsets[1:][None]).sum(-1)       # the token's sequence
    live = torch.ones(n, device="cuda") if s.mask is None else s.mask.float()
    u = s.logits if c["gating"] == 1 else -torch.log1p(torch.exp(-s.logits.abs())) + s.logits.clamp(max=0.0)
    p = torch.exp(u - u.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    p = p * live[:, None]
    tokens = torch.zeros(q, device="cuda").index_add_(0, of, live)
    per = tokens.clamp(min=1.0)
    counts = torch.zeros(q * e, dtype=torch.int32, device="cuda")
    counts.scatter_add_(0, (of[:, None] * e + s.ids.long()).flatten(), live.to(torch.int32)[:, None].expand(n, k).flatten())
    counts = counts.view(q, e)
    prob = torch.zeros(q, e, dtype=torch.float64, device="cuda").index_add_(0, of, p.double())
    prob = (prob / per[:, None]).float()
    factor = s.coef * e / k / (tokens > 0).sum().clamp(min=1)
    loss = (factor * (counts * prob).sum(-1) / per).sum()
    weight = counts * (factor / per ** 2)[:, None]
    row = weight[of]
    grad = p * (row - (p * row).sum(-1, keepdim=True))
    if c["gating"] == 2:
        grad = grad / (1.0 + torch.exp(s.logits))
    return {"loss": loss, "counts": counts, "prob": prob, "grad": grad}


# ---- the definitions in 64 bits ----

def _exact_product(x, w, w_scale):
    """rows of 64-bit values through the 8-bit product"""
    top = x.abs().max(-1, keepdim=True).values
    q = torch.round(127.0 * x / torch.where(top > 0, top, torch.ones_like(top)))
    return (q @ w.double().T) * (top / 127.0) * w_scale.double()


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "linear":
        return _exact_product(s.x.double(), s.w, s.w_scale)
    if case["kind"] == "experts":
        out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            t, j = (s.ids == e).nonzero(as_tuple=True)
            if t.numel():
                x = s.x[t].double()
                g, u = _exact_product(x, s.gate[e], s.gate_scale[e]), _exact_product(x, s.up[e], s.up_scale[e])
                y = _exact_product(g * torch.sigmoid(g) * u, s.down[e], s.down_scale[e])
                out.index_add_(0, t, y * s.weights[t, j].double()[:, None])
        return out
    score = torch.softmax(s.logits.double(), -1)
    if case["gating"] == 2:
        score = torch.sigmoid(s.logits.double())
        score = score / score.sum(-1, keepdim=True)
    e, k, ends = case["experts"], case["topk"], s.offsets.tolist()
    kept = torch.ones(case["tokens"], dtype=torch.bool, device="cuda") if s.mask is None else s.mask
    spans = [kept.new_zeros(kept.shape).index_fill_(0, torch.arange(a, b, device="cuda"), True) & kept for a, b in zip(ends, ends[1:])]
    filled = sum(bool(m.any()) for m in spans)
    loss, counts, prob, grad = 0.0, [], [], torch.zeros_like(score)
    for m in spans:
        t = int(m.sum())
        c = torch.bincount(s.ids[m].flatten().long(), minlength=e).double()
        mean = score[m].sum(0) / max(t, 1)
        counts.append(c)
        prob.append(mean)
        if t:
            f = s.coef * e / (k * t * filled) * c
            loss = loss + (f * mean).sum()
            rows = score[m] * (f / t - (score[m] * f / t).sum(-1, keepdim=True))
            grad[m] = rows * (1.0 - torch.sigmoid(s.logits[m].double())) if case["gating"] == 2 else rows
    return {"loss": torch.as_tensor(loss, dtype=torch.float64), "counts": torch.stack(counts).int(), "prob": torch.stack(prob), "grad": grad}
