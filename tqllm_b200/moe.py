"""Host-side harness over the C ABI: torch tensors own the device memory, every computation goes through libb2moe.so.

This is the Python mirror used by the tests and the benchmark; tqLLM itself binds the same C ABI from C++ through the
adapter in tqllm_b200/adapter/. Names follow the reference's: banks of stacked experts, routing ids / weights, the
dispatch plan (counts, offsets, permutation), the layer forward.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import capi
from .capi import check, lib

_DT = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
_INT = (1 << 31) - 1                       # the C ABI's int32: ctypes would take a larger number's low bits


def _stream() -> int:
    """handle of the current device's current stream (torch.cuda.current_stream().cuda_stream makes a Stream object for it: 3.3 us a call)"""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream_of(t: torch.Tensor, *others: torch.Tensor | None, banks: tuple = ()) -> int:
    """the current stream, for tensors and banks that are all on the current device (a launch there on another one's memory would fault)"""
    dev = t.get_device()
    if dev >= 0 and dev == torch._C._cuda_getDevice():
        for o in others:
            if o is not None and o.get_device() != dev:
                break
        else:
            for b in banks:
                if b is not None and b.index != dev:
                    break
            else:
                return torch._C._cuda_getCurrentRawStream(dev)
    raise capi.B2moeError(capi.ERR_CUDA, "tensors on the current CUDA device are wanted")


class DeviceBank:
    """One stacked expert matrix [experts * rows][cols] in bank layout on the device (`index`: the device's, asked for once; -1 for host memory)."""

    def __init__(self, type_id: int, raw: torch.Tensor, experts: int, rows: int, cols: int):
        assert raw.is_cuda and raw.dtype == torch.uint8
        if raw.numel() != experts * lib.b2moe_raw_bytes(type_id, rows, cols) or raw.numel() == 0:
            raise capi.B2moeError(capi.ERR_SHAPE, "DeviceBank: raw byte count does not match the shape")
        self.type, self.experts, self.rows, self.cols = type_id, experts, rows, cols
        self.data = torch.empty(experts * lib.b2moe_bank_bytes(type_id, rows, cols), dtype=torch.uint8, device=raw.device)
        aux_bytes = lib.b2moe_bank_aux_bytes(type_id, rows, cols)
        self.aux = torch.empty(experts * aux_bytes // 4, dtype=torch.float32, device=raw.device) if aux_bytes else None
        check(lib.b2moe_bank_load(type_id, raw.data_ptr(), experts, rows, cols, self.data.data_ptr(), _ptr(self.aux), _stream()),
              "b2moe_bank_load")
        self.c, self.index = capi.Bank(self.data.data_ptr(), _ptr(self.aux), type_id, experts, rows, cols), self.data.get_device()

    @classmethod
    def from_packed(cls, type_id: int, data, aux, experts: int, rows: int, cols: int, device="cuda"):
        """a bank that was packed on the host (b2moe_bank_pack_host, b2moe_gguf_expert_bank): one upload, no device repack"""
        self = cls.__new__(cls)
        self.type, self.experts, self.rows, self.cols = type_id, experts, rows, cols
        if len(data) != lib.b2moe_bank_bytes(type_id, experts * rows, cols):
            raise capi.B2moeError(capi.ERR_SHAPE, "DeviceBank.from_packed: byte count does not match the shape")
        self.data = torch.as_tensor(data).to(device)
        self.aux = None if aux is None else torch.as_tensor(aux).to(device)
        self.c, self.index = capi.Bank(self.data.data_ptr(), _ptr(self.aux), type_id, experts, rows, cols), self.data.get_device()
        return self

    @classmethod
    def from_int8(cls, data: torch.Tensor, scale: torch.Tensor, experts: int = 1):
        """A bank of 8-bit rows over the caller's arrays, which it keeps and does not copy: data int8 [experts * rows, cols] (or
        [experts, rows, cols]), scale float32 with one value a row."""
        rows, cols = data.shape[-2] if data.dim() == 3 else data.shape[0] // experts, data.shape[-1]
        experts = data.shape[0] if data.dim() == 3 else experts
        if data.dtype != torch.int8 or scale.dtype != torch.float32 or not data.is_contiguous() or not scale.is_contiguous():
            raise capi.B2moeError(capi.ERR_FORMAT, "DeviceBank.from_int8: contiguous int8 rows and float32 scales are wanted")
        if data.numel() != experts * rows * cols or scale.numel() != experts * rows or data.device != scale.device:
            raise capi.B2moeError(capi.ERR_SHAPE, "DeviceBank.from_int8: a scale for each row is wanted, on the same device")
        if max(experts, rows, cols) > _INT:
            raise capi.B2moeError(capi.ERR_SHAPE, "DeviceBank.from_int8: experts, rows and columns are 32-bit numbers")
        self = cls.__new__(cls)
        self.type, self.experts, self.rows, self.cols = capi.I8, experts, rows, cols
        self.data, self.aux = data, scale
        self.c, self.index = capi.Bank(data.data_ptr(), scale.data_ptr(), capi.I8, experts, rows, cols), data.get_device()
        return self

    @classmethod
    def from_float(cls, w: torch.Tensor):
        """floating-point weights [experts, rows, cols] (or [rows, cols]) quantised to a bank of 8-bit rows (b2moe_quantize_rows)"""
        q, scale = quantize_rows(w.reshape(-1, w.shape[-1]))
        return cls.from_int8(q.view(w.shape), scale.view(w.shape[:-1]), 1)

    def dequant(self) -> torch.Tensor:
        stream = _stream_of(self.data, self.aux)
        out = torch.empty(self.experts * self.rows, self.cols, dtype=torch.float32, device=self.data.device)
        check(lib.b2moe_dequant_dump(C.byref(self.c), out.data_ptr(), stream), "b2moe_dequant_dump")
        return out


def router(router_w, x, shared_gate=None, ld=None):
    n, h = x.shape
    e = router_w.shape[0]
    ld = ld or e + 1
    logits = torch.zeros(n, ld, dtype=torch.float32, device=x.device)
    check(lib.b2moe_router(router_w.data_ptr(), _ptr(shared_gate), x.data_ptr(), _DT[x.dtype], logits.data_ptr(), ld, h, e, n, _stream()),
          "b2moe_router")
    return logits


def topk_softmax(logits, experts, k, scale=0.0, shared=False):
    n, ld = logits.shape
    ids = torch.empty(n, k, dtype=torch.int32, device=logits.device)
    w = torch.empty(n, k, dtype=torch.float32, device=logits.device)
    sw = torch.empty(n, dtype=torch.float32, device=logits.device) if shared else None
    check(lib.b2moe_topk_softmax(logits.data_ptr(), ld, ids.data_ptr(), w.data_ptr(), _ptr(sw), experts, k, n, scale, _stream()),
          "b2moe_topk_softmax")
    return ids, w, sw



def topk_softmax2(logits, logits2, experts, k, scale=0.0, shared=False):
    """Two routings of the same tokens in one launch (the reference's moe_topk2): returns ((ids, w, sw), (ids2, w2, sw2))."""
    n, ld = logits.shape
    assert logits2.shape == logits.shape
    out = []
    for _ in range(2):
        out.append((torch.empty(n, k, dtype=torch.int32, device=logits.device), torch.empty(n, k, dtype=torch.float32, device=logits.device),
                    torch.empty(n, dtype=torch.float32, device=logits.device) if shared else None))
    (i1, w1, s1), (i2, w2, s2) = out
    check(lib.b2moe_topk_softmax2(logits.data_ptr(), i1.data_ptr(), w1.data_ptr(), _ptr(s1), logits2.data_ptr(), i2.data_ptr(), w2.data_ptr(),
                                  _ptr(s2), ld, experts, k, n, scale, _stream()), "b2moe_topk_softmax2")
    return out

def route_sigmoid(logits, experts, k, bias=None, norm=True, scale=0.0):
    n, ld = logits.shape
    ids = torch.empty(n, k, dtype=torch.int32, device=logits.device)
    w = torch.empty(n, k, dtype=torch.float32, device=logits.device)
    check(lib.b2moe_route_sigmoid(logits.data_ptr(), ld, _ptr(bias), ids.data_ptr(), w.data_ptr(), experts, k, int(norm), scale, n,
                                  _stream()), "b2moe_route_sigmoid")
    return ids, w


def quantize_rows(x: torch.Tensor):
    """(q int8 [n, k], scale float32 [n]) of the rows of x (b2moe_quantize_rows); x may be rows of a wider matrix"""
    n, k = x.shape
    ldx, one = x.stride()
    if one != 1 and k > 1:
        raise capi.B2moeError(capi.ERR_SHAPE, "quantize_rows: the values of a row have to be neighbours")
    if max(n, k) > _INT:
        raise capi.B2moeError(capi.ERR_SHAPE, "quantize_rows: rows and columns are 32-bit numbers")
    stream = _stream_of(x)
    q = torch.empty(n, k, dtype=torch.int8, device=x.device)
    scale = torch.empty(n, dtype=torch.float32, device=x.device)
    check(lib.b2moe_quantize_rows(x.data_ptr(), _DT[x.dtype], ldx if n > 1 else k, n, k, q.data_ptr(), k, scale.data_ptr(), stream), "b2moe_quantize_rows")
    return q, scale


def linear_i8(q: torch.Tensor, scale: torch.Tensor, bank: DeviceBank, out_dtype=torch.bfloat16, out: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """y [n, rows] = (q . w) * scale[t] * bank scale[r] of 8-bit rows (b2moe_linear_i8); q and out may be rows of wider matrices. A launch that gives up a bounded
    wait leaves NaN in what it did not finish, and a nonzero value in `status` where that is given"""
    n, k = q.shape
    ldq, one = q.stride()
    ldy = rows = bank.rows
    if q.dtype is not torch.int8 or k != bank.cols or scale.dtype is not torch.float32 or scale.numel() != n or not scale.is_contiguous():
        raise capi.B2moeError(capi.ERR_SHAPE, "linear_i8: int8 rows of the bank's columns and a float32 scale for each are wanted")
    if one != 1 and k > 1:
        raise capi.B2moeError(capi.ERR_SHAPE, "linear_i8: the values of a row have to be neighbours")
    if n > _INT:
        raise capi.B2moeError(capi.ERR_SHAPE, "linear_i8: the number of rows is a 32-bit number")
    if status is not None and (status.dtype is not torch.int32 or status.numel() < 1):
        raise capi.B2moeError(capi.ERR_SHAPE, "linear_i8: the status is an int32 word")
    if out is not None:
        if out.shape != (n, rows) or (out.stride(1) != 1 and rows > 1):
            raise capi.B2moeError(capi.ERR_SHAPE, "linear_i8: an output [n, rows] with contiguous rows is wanted")
        out_dtype = out.dtype
        ldy = out.stride(0) if n > 1 else rows
    stream = _stream_of(q, scale, out, status, banks=(bank,))
    if out is None:
        out = torch.empty(n, rows, dtype=out_dtype, device=q.device)
    check(lib.b2moe_linear_i8(q.data_ptr(), ldq if n > 1 else k, scale.data_ptr(), C.byref(bank.c), n, out.data_ptr(), _DT[out_dtype], ldy, _ptr(status), stream), "b2moe_linear_i8")
    return out


class Balance(NamedTuple):
    """what b2moe_balance_loss writes: loss (a scalar), counts and prob [sequences, experts], tokens [sequences + 1]"""
    loss: torch.Tensor
    counts: torch.Tensor
    prob: torch.Tensor
    tokens: torch.Tensor


def _balance_args(logits, experts, mask, offsets):
    n, cols = logits.shape
    ld, one = logits.stride()
    if logits.dtype is not torch.float32 or cols < experts or (one != 1 and experts > 1):
        raise capi.B2moeError(capi.ERR_SHAPE, "balance loss: float32 logits with contiguous rows of at least as many columns as experts are wanted")
    if max(n, ld if n > 1 else cols) > _INT:                           # (experts are no more than the columns)
        raise capi.B2moeError(capi.ERR_SHAPE, "balance loss: tokens, columns and the row stride of the logits are 32-bit numbers")
    if mask is not None and (mask.numel() != n or mask.dtype not in (torch.bool, torch.uint8) or not mask.is_contiguous()):
        raise capi.B2moeError(capi.ERR_SHAPE, "balance loss: the mask has a byte for each token")
    if offsets is None:
        return n, ld if n > 1 else cols, 1
    sequences = offsets.numel() - 1
    if offsets.dtype is not torch.int32 or sequences < 1 or sequences > _INT or not offsets.is_contiguous():
        raise capi.B2moeError(capi.ERR_SHAPE, "balance loss: the offsets are int32, one more than sequences")
    return n, ld if n > 1 else cols, sequences


def balance_loss(logits, ids, experts, coef, gating=capi.SOFTMAX, mask=None, offsets=None) -> Balance:
    """The router's balance loss over logits [n, >= experts] and the ids [n, topk] that were routed (b2moe_balance_loss)."""
    n, ld, seqs = _balance_args(logits, experts, mask, offsets)
    tokens, topk = ids.shape
    if tokens != n or ids.dtype is not torch.int32 or not ids.is_contiguous():
        raise capi.B2moeError(capi.ERR_SHAPE, "balance loss: contiguous int32 ids [n, topk] are wanted")
    stream = _stream_of(logits, ids, mask, offsets)
    new, ints = logits.new_empty, ids.new_empty
    out = Balance(new(()), ints((seqs, experts)), new((seqs, experts)), ints(seqs + 1))
    size = lib.b2moe_balance_workspace_bytes(experts, n, seqs)
    ws = new(max(4, size // 4))
    check(lib.b2moe_balance_loss(gating, logits.data_ptr(), ld, ids.data_ptr(), topk, _ptr(mask), _ptr(offsets), seqs, experts, n, coef, out.loss.data_ptr(),
                                 out.counts.data_ptr(), out.prob.data_ptr(), out.tokens.data_ptr(), ws.data_ptr(), size, stream), "b2moe_balance_loss")
    return out


def balance_loss_backward(logits, saved: Balance, topk, coef, gating=capi.SOFTMAX, mask=None, offsets=None, grad_loss=None, out=None):
    """The gradient of the balance loss on the logits, [n, experts]; into `out` (rows of at least `experts` columns) it is added."""
    counted, experts = saved.counts.shape
    n, ld, seqs = _balance_args(logits, experts, mask, offsets)
    if counted != seqs or saved.tokens.shape != (seqs + 1,) or saved.counts.dtype is not torch.int32 or saved.tokens.dtype is not torch.int32 or not (
            saved.counts.is_contiguous() and saved.tokens.is_contiguous()):
        raise capi.B2moeError(capi.ERR_SHAPE, "balance loss: int32 counts and tokens of the same sequences are wanted, as the loss leaves them")
    if grad_loss is not None and (grad_loss.dtype is not torch.float32 or grad_loss.numel() != 1):
        raise capi.B2moeError(capi.ERR_SHAPE, "balance loss: the loss's gradient is one float32")
    grad, ldg = out, experts
    if grad is not None:
        if grad.dtype is not torch.float32 or grad.shape[0] != n or grad.shape[1] < experts or (grad.stride(1) != 1 and experts > 1):
            raise capi.B2moeError(capi.ERR_SHAPE, "balance loss: the gradient has float32 rows like the logits")
        ldg = grad.stride(0) if n > 1 else grad.shape[1]
        if ldg > _INT:
            raise capi.B2moeError(capi.ERR_SHAPE, "balance loss: the row stride of the gradient is a 32-bit number")
    stream = _stream_of(logits, saved.counts, saved.tokens, mask, offsets, grad_loss, out)
    if grad is None:
        grad = logits.new_empty((n, experts))
    check(lib.b2moe_balance_loss_backward(gating, logits.data_ptr(), ld, topk, _ptr(mask), _ptr(offsets), seqs, experts, n, coef, saved.counts.data_ptr(),
                                          saved.tokens.data_ptr(), _ptr(grad_loss), grad.data_ptr(), ldg, int(out is not None), stream), "b2moe_balance_loss_backward")
    return grad


def count_ids(ids: torch.Tensor, counts: torch.Tensor) -> torch.Tensor:
    """counts[e] += occurrences of e in ids (the reference's moe_count): counts is an int64 device tensor [experts]"""
    assert counts.dtype == torch.int64 and ids.dtype == torch.int32
    check(lib.b2moe_count(ids.data_ptr(), counts.data_ptr(), ids.numel(), counts.numel(), _stream()), "b2moe_count")
    return counts


def place_experts(counts, ranks: int):
    """Load-aware placement from a routing histogram: (order, rank_load) with order[r * per + i] = the expert in slot i of
    rank r (host arithmetic, b2moe_place_experts); feed `order` to synth.permute_experts or the loader's equivalent."""
    import numpy as np
    c = np.ascontiguousarray(np.asarray(counts.cpu() if hasattr(counts, "cpu") else counts), dtype=np.uint64)
    order = np.empty(c.size, np.int32)
    load = np.empty(ranks, np.uint64)
    check(lib.b2moe_place_experts(c.ctypes.data, c.size, ranks, order.ctypes.data, load.ctypes.data), "b2moe_place_experts")
    return order, load


class Plan:
    """Device dispatch plan with views of its arrays."""

    def __init__(self, experts: int, n: int, topk: int, shared_tokens: int, device):
        self.experts, self.n, self.topk, self.shared_tokens = experts, n, topk, shared_tokens
        v = capi.PlanView()
        lib.b2moe_plan_view_of(experts, n * topk, shared_tokens, C.byref(v))
        self.view = v
        self.buf = torch.zeros(v.total, dtype=torch.int32, device=device)

    @property
    def n_active(self): return int(self.buf[0])
    @property
    def counts(self): return self.buf[self.view.counts:self.view.counts + self.experts + 1]
    @property
    def offsets(self): return self.buf[self.view.offsets:self.view.offsets + self.experts + 2]
    @property
    def active(self): return self.buf[self.view.active:self.view.active + self.experts + 1]
    @property
    def perm(self): return self.buf[self.view.perm:self.view.passes]
    @property
    def passes(self): return self.buf[self.view.passes:self.view.total]


def dispatch(ids: torch.Tensor, experts: int, shared_tokens: int = 0) -> Plan:
    n, k = ids.shape
    plan = Plan(experts, n, k, shared_tokens, ids.device)
    wsb = lib.b2moe_dispatch_workspace_bytes(experts, n * k)
    ws = torch.empty(max(wsb, 16), dtype=torch.uint8, device=ids.device)
    check(lib.b2moe_dispatch(ids.data_ptr(), n, k, experts, shared_tokens, plan.buf.data_ptr(), ws.data_ptr(), ws.numel(), _stream()),
          "b2moe_dispatch")
    return plan


def plan_to_groups(plan: Plan):
    counts = torch.zeros(plan.experts, dtype=torch.int32, device=plan.buf.device)
    groups = torch.full((plan.experts, plan.n), -1, dtype=torch.int32, device=plan.buf.device)
    check(lib.b2moe_plan_to_groups(plan.buf.data_ptr(), plan.n, plan.topk, plan.experts, counts.data_ptr(), groups.data_ptr(), _stream()),
          "b2moe_plan_to_groups")
    return counts, groups


def _scratch(nbytes: int, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _bref(b: DeviceBank | None):
    return C.byref(b.c) if b is not None else None


def expert_gateup_swiglu(gate, up, x, plan: Plan, sh_gate=None, sh_up=None, act: torch.Tensor | None = None):
    """act [assignments, ff]; a buffer that is given keeps the rows of skipped assignments, without one they are zeros"""
    total = plan.n * plan.topk + plan.shared_tokens
    stream = _stream_of(x, plan.buf, act, banks=(gate, up, sh_gate, sh_up))
    act = torch.zeros(total, gate.rows, dtype=torch.float32, device=x.device) if act is None else act
    assert act.dtype == torch.float32 and act.shape == (total, gate.rows) and act.is_contiguous()
    # room for a row per assignment: the grouped GEMM reads the rows of an expert as boxes then and does not gather them
    ws = _scratch(lib.b2moe_expert_slot_workspace_bytes(_bref(gate), total, _DT[x.dtype]), x.device)
    check(lib.b2moe_expert_gateup_swiglu(_bref(gate), _bref(up), _bref(sh_gate), _bref(sh_up), x.data_ptr(), _DT[x.dtype],
                                         plan.buf.data_ptr(), plan.n, plan.topk, plan.shared_tokens, act.data_ptr(),
                                         _ptr(ws), 0 if ws is None else ws.numel(), stream), "b2moe_expert_gateup_swiglu")
    return act


def expert_down(down, act, plan: Plan, sh_down=None, y: torch.Tensor | None = None):
    """y [assignments, hidden]; a buffer that is given keeps the rows of skipped assignments, without one they are zeros"""
    stream = _stream_of(act, plan.buf, y, banks=(down, sh_down))
    y = torch.zeros(act.shape[0], down.rows, dtype=torch.float32, device=act.device) if y is None else y
    assert y.dtype == torch.float32 and y.shape == (act.shape[0], down.rows) and y.is_contiguous()
    ws = _scratch(lib.b2moe_expert_slot_workspace_bytes(_bref(down), act.shape[0], capi.F32), act.device)
    check(lib.b2moe_expert_down(_bref(down), _bref(sh_down), act.data_ptr(), plan.buf.data_ptr(), plan.n, plan.topk,
                                plan.shared_tokens, y.data_ptr(), _ptr(ws), 0 if ws is None else ws.numel(), stream),
          "b2moe_expert_down")
    return y


def combine(y, weights, n, topk, hidden, shared_tokens=0, shared_weights=None, ids=None, out_dtype=torch.float32):
    out = torch.empty(n, hidden, dtype=out_dtype, device=y.device)
    check(lib.b2moe_combine(y.data_ptr(), _ptr(ids), weights.data_ptr(), _ptr(shared_weights), n, topk, hidden, shared_tokens,
                            out.data_ptr(), _DT[out_dtype], _stream()), "b2moe_combine")
    return out


class MoeLayer:
    """A resident MoE layer: router weight, expert banks (+ shared expert), and a workspace sized for `max_tokens`."""

    def __init__(self, shape, router_w, raw, shared_raw=None, sel_bias=None, shared_gate_vec=None, experts=None,
                 device="cuda", iq3s_layout="codes"):
        """iq3s_layout: "codes" loads IQ3_S blocks into the 4-bit-code bank layout (capi.IQ3_S_X4: 21.8 % more HBM, decode
        kernels without a codebook lookup), "gguf" into the layout of the GGUF block size."""
        E = experts or shape.experts
        self.shape, self.experts, self.device = shape, E, torch.device(device)
        H, F = shape.hidden, shape.ff
        dev = lambda t: None if t is None else t.to(self.device).contiguous()
        self.router_w, self.sel_bias, self.shared_gate_vec = dev(router_w), dev(sel_bias), dev(shared_gate_vec)
        assert iq3s_layout in ("codes", "gguf")
        tg, tu, td = (capi.IQ3_S_X4 if (t == capi.IQ3_S and iq3s_layout == "codes") else t for t in shape.types)
        self.gate = DeviceBank(tg, dev(raw[0]), E, F, H)
        self.up = DeviceBank(tu, dev(raw[1]), E, F, H)
        self.down = DeviceBank(td, dev(raw[2]), E, H, F)
        self.sh = None
        if shared_raw is not None:
            self.sh = (DeviceBank(tg, dev(shared_raw[0]), 1, F, H), DeviceBank(tu, dev(shared_raw[1]), 1, F, H),
                       DeviceBank(td, dev(shared_raw[2]), 1, H, F))
        self._finish()

    def _finish(self):
        shape, E, H, F = self.shape, self.experts, self.shape.hidden, self.shape.ff
        L = capi.Layer()
        L.hidden, L.experts, L.topk, L.ff = H, E, shape.topk, F
        L.gating, L.norm, L.scale, L.has_shared = shape.gating, int(shape.norm), shape.scale, int(self.sh is not None)
        L.router_w, L.sel_bias, L.shared_gate_vec = _ptr(self.router_w), _ptr(self.sel_bias), _ptr(self.shared_gate_vec)
        L.gate, L.up, L.down = self.gate.c, self.up.c, self.down.c
        if self.sh:
            L.sh_gate, L.sh_up, L.sh_down = self.sh[0].c, self.sh[1].c, self.sh[2].c
        self.c = L
        self.ws, self.ws_view, self.ws_tokens = None, None, 0

    @classmethod
    def from_gguf(cls, path, shape, layer_index=0, first_expert=0, experts=None, device="cuda", iq3s_layout="codes"):
        """Experts [first_expert, first_expert + experts) of layer `layer_index` of a GGUF checkpoint (tensor names
        blk.N.ffn_{gate,up,down}_exps.weight, router blk.N.ffn_gate_inp.weight, optional blk.N.ffn_{gate,up,down}_shexp.weight):
        the banks are packed on the host by the library's reader and uploaded once."""
        import numpy as np
        from . import gguf
        pre = f"blk.{layer_index}."
        with gguf.GgufExperts(path) as g:
            names = g.names()
            t, (h, e_all, _), off, _ = g.tensor(pre + "ffn_gate_inp.weight")
            assert t == 0 and h == shape.hidden, "router must be an F32 [hidden, experts] tensor"
            E = experts or e_all - first_expert
            router = np.array(np.memmap(path, np.float32, "r", off, (e_all, h))[first_expert:first_expert + E])
            codes = iq3s_layout == "codes"
            banks = [g.expert_bank(pre + f"ffn_{m}_exps.weight", first_expert, E, codes) for m in ("gate", "up", "down")]
            shared = None
            if pre + "ffn_gate_shexp.weight" in names:
                shared = [g.expert_bank(pre + f"ffn_{m}_shexp.weight", 0, 1, codes) for m in ("gate", "up", "down")]
        self = cls.__new__(cls)
        self.shape, self.experts, self.device = shape, E, torch.device(device)
        self.router_w, self.sel_bias, self.shared_gate_vec = torch.from_numpy(router).to(device), None, None
        mk = lambda b, n: DeviceBank.from_packed(b[0], b[3], b[4], n, b[1], b[2], device)
        self.gate, self.up, self.down = (mk(b, E) for b in banks)
        self.sh = tuple(mk(b, 1) for b in shared) if shared else None
        self._finish()
        return self

    @classmethod
    def from_banks(cls, shape, router_w, banks, shared_banks=None, sel_bias=None, shared_gate_vec=None):
        """A layer over finished banks (DeviceBank: gate, up, down, of any types, 8-bit ones among them) that it keeps, with router_w [experts, hidden],
        sel_bias [experts] and shared_gate_vec [hidden] in contiguous float32; shape.types is not looked at"""
        for t, dims in ((router_w, (banks[0].experts, shape.hidden)), (sel_bias, (banks[0].experts,)), (shared_gate_vec, (shape.hidden,))):
            if t is not None and (t.dtype is not torch.float32 or tuple(t.shape) != dims or not t.is_contiguous()):
                raise capi.B2moeError(capi.ERR_SHAPE, "MoeLayer.from_banks: contiguous float32 router weights, selection bias and shared gate of the layer's sizes are wanted")
        _stream_of(router_w, sel_bias, shared_gate_vec, banks=(*banks, *(shared_banks or ())))
        self = cls.__new__(cls)
        self.shape, self.experts, self.device = shape, banks[0].experts, router_w.device
        self.router_w, self.sel_bias, self.shared_gate_vec = router_w, sel_bias, shared_gate_vec
        self.gate, self.up, self.down = banks
        self.sh = tuple(shared_banks) if shared_banks is not None else None
        self._finish()
        return self

    @classmethod
    def from_synth(cls, layer, device="cuda", experts=None, shared_gate_vec=None, iq3s_layout="codes"):
        return cls(layer.shape, layer.router_w, layer.raw, layer.shared_raw, layer.sel_bias, shared_gate_vec,
                   experts=experts or layer.router_w.shape[0], device=device, iq3s_layout=iq3s_layout)

    def reserve(self, n: int):
        if self.ws is not None and self.ws_tokens == n:
            return
        v = capi.LayerWs()
        check(lib.b2moe_layer_workspace(C.byref(self.c), n, C.byref(v)), "b2moe_layer_workspace")
        self.ws = torch.zeros(v.total, dtype=torch.uint8, device=self.device)
        self.ws_view, self.ws_tokens = v, n

    def forward(self, x: torch.Tensor, out: torch.Tensor | None = None, out_dtype=torch.float32, residual: torch.Tensor | None = None) -> torch.Tensor:
        """out = layer(x), or residual + layer(x) when a residual [n][hidden] of the output's dtype is given (it may be `out`)"""
        n = x.shape[0]
        stream = _stream_of(self.router_w, x, out, residual)
        self.reserve(n)
        if out is None:
            out = torch.empty(n, self.shape.hidden, dtype=out_dtype if residual is None else residual.dtype, device=self.device)
        if residual is None:
            check(lib.b2moe_layer_forward(C.byref(self.c), x.data_ptr(), _DT[x.dtype], n, out.data_ptr(), _DT[out.dtype],
                                          self.ws.data_ptr(), self.ws.numel(), stream), "b2moe_layer_forward")
        else:
            assert residual.dtype == out.dtype and residual.shape == out.shape
            check(lib.b2moe_layer_forward_residual(C.byref(self.c), x.data_ptr(), _DT[x.dtype], n, residual.data_ptr(), out.data_ptr(),
                                                   _DT[out.dtype], self.ws.data_ptr(), self.ws.numel(), stream), "b2moe_layer_forward_residual")
        return out

    def artefacts(self) -> dict:
        """The routing / dispatch intermediates of the last forward, read back from the workspace."""
        v, n, k, E = self.ws_view, self.ws_tokens, self.shape.topk, self.experts

        def view(off, count, dtype):
            return self.ws[off:off + count * 4].view(dtype)

        pv = capi.PlanView()
        sh = n if self.sh else 0
        lib.b2moe_plan_view_of(E, n * k, sh, C.byref(pv))
        plan = view(v.plan, pv.total, torch.int32)
        return dict(
            logits=view(v.logits, n * (E + 1), torch.float32).reshape(n, E + 1),
            ids=view(v.ids, n * k, torch.int32).reshape(n, k),
            weights=view(v.weights, n * k, torch.float32).reshape(n, k),
            shared_weights=view(v.shared_weights, n, torch.float32),
            n_active=int(plan[0]),
            counts=plan[pv.counts:pv.counts + E + 1], offsets=plan[pv.offsets:pv.offsets + E + 2],
            active=plan[pv.active:pv.active + E + 1], perm=plan[pv.perm:pv.passes], passes=plan[pv.passes:pv.total],
            status=int(plan[3]),
            act=view(v.act, (n * k + sh) * self.shape.ff, torch.float32).reshape(n * k + sh, self.shape.ff),
            y=view(v.y, (n * k + sh) * self.shape.hidden, torch.float32).reshape(n * k + sh, self.shape.hidden),
        )
