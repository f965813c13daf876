"""Python mirror of the reference's operator API for the MoE expert path, over libtsx_moe.so.

Names and argument meanings follow TinyStrata's C++ headers (include/strata/kernels/iq_kernels.hpp,
native_mmvq.hpp, native_router.hpp, include/strata/prefill/moe_mmq.hpp); buffers are torch tensors in device
memory (PyTorch is only the allocator and the stream here), and every call enqueues on the current stream.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from ._lib import (BF16, F16, F32, IQ3_S, IQ3_XXS, Q4_K, Q8_0, AdapterArgs, ExpertLayout, MmqProduct, MmvqIds, MmvqSlots,
                   RouterArgs, check, lib)

WEIGHT_TYPES = (Q8_0, Q4_K, IQ3_XXS, IQ3_S)
Q8_1_BLOCK_BYTES = 36


def _p(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("device tensors only")
    return t.data_ptr()


def _stream(stream=None) -> int:
    if stream is not None:
        return stream.cuda_stream
    # the handle alone: torch.cuda.current_stream() makes an object first, 2.6 us of a call's 10
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


PLAIN_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def _expect(what: str, name: str, t: torch.Tensor | None, shape, dtype, like: torch.Tensor | None = None,
            rows: bool = False) -> None:
    """Refuses a tensor of another type, shape or device than the call takes (None stands for an absent one); `rows`:
    rows may lie further apart than their length, else the tensor is dense."""
    if t is None:
        return
    if t.dtype != dtype:
        raise ValueError(f"{what}: {name} is {t.dtype}, not {dtype}")
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if like is not None and t.device != like.device:
        raise ValueError(f"{what}: {name} is on {t.device}, not {like.device}")
    if t.is_contiguous():
        return
    if rows:
        if t.numel() and ((t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1])):
            raise ValueError(f"{what}: {name}'s rows are not dense (strides {t.stride()})")
    else:
        raise ValueError(f"{what}: {name} is not contiguous")


def _ld(t: torch.Tensor | None) -> int:
    """Values between a matrix's rows (of a single row: its length)."""
    return 0 if t is None else t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _launch(what: str, fn, like: torch.Tensor, stream, *args) -> None:
    """fn(*args, stream) on like's device: on its current stream unless one is given."""
    if not like.is_cuda:
        raise ValueError("device tensors only")
    if like.device.index == torch.cuda.current_device():
        check(fn(*args, _stream(stream)), what)
        return
    with torch.cuda.device(like.device):
        check(fn(*args, _stream(stream)), what)


# ------------------------------------------------------------------ formats
def iq_supported(ggml_type: int) -> bool:
    return ggml_type in WEIGHT_TYPES


def iq_row_bytes(ggml_type: int, n: int) -> int:
    return lib().tsx_moe_row_bytes(ggml_type, n)


def native_expert_supported(gu_type: int, d_type: int, n_embd: int, n_ff: int) -> bool:
    return bool(lib().tsx_moe_expert_supported(gu_type, d_type, n_embd, n_ff))


def native_expert_layout(gu_type: int, d_type: int, n_embd: int, n_ff: int) -> ExpertLayout:
    L = ExpertLayout()
    check(lib().tsx_moe_expert_layout(gu_type, d_type, n_embd, n_ff, C.byref(L)), "native_expert_layout")
    return L


def native_expert_scratch_bytes(cap_entries: int, n_ff: int) -> int:
    return lib().tsx_moe_expert_scratch_bytes(cap_entries, n_ff)


def scratch_hq_offset(cap_entries: int, n_ff: int) -> int:
    return lib().tsx_moe_expert_scratch_hq_offset(cap_entries, n_ff)


# ------------------------------------------------------------------ activations
def quantize_q8_1_rows(x: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """x [rows, cols] float32 -> Q8_1 blocks, uint8 [rows, cols/32*36]."""
    rows, cols = x.shape
    if out is None:
        out = torch.empty((rows, cols // 32 * Q8_1_BLOCK_BYTES), dtype=torch.uint8, device=x.device)
    check(lib().tsx_moe_quantize_q8_1(_p(x), rows, cols, _p(out), _stream(stream)), "quantize_q8_1_rows")
    return out


def native_swiglu_quantize_q8_1(gate: torch.Tensor, up: torch.Tensor, out: torch.Tensor | None = None, stream=None):
    n = gate.numel()
    if out is None:
        out = torch.empty(n // 32 * Q8_1_BLOCK_BYTES, dtype=torch.uint8, device=gate.device)
    check(lib().tsx_moe_swiglu_quantize_q8_1(_p(gate), _p(up), n, _p(out), _stream(stream)), "native_swiglu_quantize_q8_1")
    return out


# ------------------------------------------------------------------ decode
def native_expert_grouped(L: ExpertLayout, grp_ptr, grp_start, n_groups, ent_dst, ent_tok, cap_groups: int,
                          cap_entries: int, x_q8_1, scratch, out, grid_groups: int = 0, stream=None) -> None:
    check(lib().tsx_moe_expert_grouped(C.byref(L), _p(grp_ptr), _p(grp_start), _p(n_groups), _p(ent_dst), _p(ent_tok),
                                       cap_groups, cap_entries, _p(x_q8_1), _p(scratch), _p(out), _stream(stream),
                                       grid_groups), "native_expert_grouped")


def iq_mmvq(ggml_type: int, w, x_q8_1, n_in: int, n_out: int, ncols: int, y=None, stream=None) -> torch.Tensor:
    """y[c][r] = W[r] . x[c] (ncols 1..8)."""
    if y is None:
        y = torch.empty((ncols, n_out), dtype=torch.float32, device=w.device)
    check(lib().tsx_moe_mmvq(ggml_type, _p(w), _p(x_q8_1), _p(y), n_in, n_out, ncols, _stream(stream)), "iq_mmvq")
    return y


native_mmvq = iq_mmvq


def mmvq_ids_supported(ggml_type: int) -> bool:
    return bool(lib().tsx_moe_mmvq_ids_supported(ggml_type))


def mmvq_ids(ggml_type: int, table: torch.Tensor, ids: torch.Tensor, offset: int, x_q8_1, x_stride: int, x_every: int,
             y: torch.Tensor, y_stride: int, count: int, n_in: int, n_out: int, stream=None) -> torch.Tensor:
    """Matrix j = table[ids[j]] + offset bytes (table: int64 device addresses), times the Q8_1 column
    x + (j / x_every) * x_stride bytes, into y + j * y_stride floats (reference lfm_native_mmvq_ids)."""
    a = MmvqIds(table=_p(table), ids=_p(ids), n_table=table.numel(), offset=offset, x=_p(x_q8_1), x_stride=x_stride,
                x_every=x_every, y=_p(y), y_stride=y_stride)
    check(lib().tsx_moe_mmvq_ids(ggml_type, C.byref(a), count, n_in, n_out, _stream(stream)), "mmvq_ids")
    return y


def mmvq_slots(ggml_type: int, ws, xs, ys, n_in: int, n_out: int, stream=None) -> None:
    """Up to 8 matrices ws[j] times their own Q8_1 column xs[j] into ys[j] (reference lfm_native_mmvq_slots)."""
    a = MmvqSlots()
    for j, (w, x, y) in enumerate(zip(ws, xs, ys)):
        a.w[j], a.x[j], a.y[j] = _p(w), _p(x), _p(y)
    check(lib().tsx_moe_mmvq_slots(ggml_type, C.byref(a), len(ws), n_in, n_out, _stream(stream)), "mmvq_slots")


def decode_layer_scratch_bytes(n_tok: int, k: int, n_ff: int) -> int:
    return lib().tsx_moe_decode_layer_scratch_bytes(n_tok, k, n_ff)


def moe_decode_layer(L: ExpertLayout, blobs, stride: int, n_expert: int, k: int, logits, x, y, ids, wts, scratch,
                     shared=None, sgate=None, sg_stride: int = 1, stream=None, norm_w=None, eps: float = 1e-6,
                     h=None, hq=None) -> None:
    """y += the whole decode MoE layer of x (1..8 tokens) in two launches (tsx_moe_decode_layer); with norm_w, also
    h = rms(y) * norm_w and (hq given) its Q8_1 image (tsx_moe_decode_layer_norm)."""
    n_tok = x.shape[0]
    # the scratch size depends on the token count (h in fp32 for one to four tokens at n_ff <= 512, as Q8_1 planes
    # otherwise): a buffer sized for another count may be too small
    need = decode_layer_scratch_bytes(n_tok, k, int(L.n_ff))
    have = scratch.numel() * scratch.element_size() if hasattr(scratch, "numel") else None
    if have is not None and have < need:
        raise ValueError(f"moe_decode_layer: scratch of {have} bytes, {n_tok} tokens x top-{k} at n_ff {int(L.n_ff)} "
                         f"need {need} (decode_layer_scratch_bytes)")
    if norm_w is None:
        check(lib().tsx_moe_decode_layer(C.byref(L), _p(blobs), stride, n_expert, k, n_tok, _p(logits), _p(x),
                                         _p(shared), _p(sgate), sg_stride, _p(y), _p(ids), _p(wts), _p(scratch),
                                         _stream(stream)), "moe_decode_layer")
        return
    check(lib().tsx_moe_decode_layer_norm(C.byref(L), _p(blobs), stride, n_expert, k, n_tok, _p(logits), _p(x),
                                          _p(shared), _p(sgate), sg_stride, _p(y), _p(ids), _p(wts), _p(norm_w), eps,
                                          _p(h), _p(hq), _p(scratch), _stream(stream)), "moe_decode_layer_norm")


# ------------------------------------------------------------------ routing
def native_router_topk(logits: torch.Tensor, k: int, ids=None, weights=None, stream=None):
    n_tok, n_expert = logits.shape
    if ids is None:
        ids = torch.empty((n_tok, k), dtype=torch.int32, device=logits.device)
    if weights is None:
        weights = torch.empty((n_tok, k), dtype=torch.float32, device=logits.device)
    check(lib().tsx_moe_router_topk(_p(logits), _p(ids), _p(weights), n_expert, k, n_tok, _stream(stream)),
          "native_router_topk")
    return ids, weights


class Router:
    """The rule by which tokens pick experts (tsx_router): softmax or sigmoid scores, a bias added for the choice alone
    (fp32 [n_expert], read at every call), the topk_group of n_group groups of experts kept (by the largest choice value
    of a group, or the sum of its two largest), weights divided by their sum (at least `floor`) when norm is set, times
    scale."""

    SCORES = {"softmax": 0, "sigmoid": 1}

    def __init__(self, n_expert: int, k: int, score: str = "softmax", bias: torch.Tensor | None = None, n_group: int = 1,
                 topk_group: int = 1, group_top: int = 1, norm: bool = True, scale: float = 1.0,
                 floor: float = 6.103515625e-5):
        if score not in self.SCORES:
            raise ValueError(f"Router: score {score!r} (softmax or sigmoid)")
        _expect("Router", "bias", bias, (n_expert,), torch.float32)
        self.n_expert, self.k, self.bias = n_expert, k, bias
        self.args = {t: RouterArgs(type=code, score=self.SCORES[score], n_expert=n_expert, k=k, n_group=n_group,
                                   topk_group=topk_group, group_top=group_top, norm=int(norm), scale=scale, floor=floor,
                                   bias=_p(bias)) for t, code in PLAIN_TYPES.items()}

    def args_for(self, what: str, logits: torch.Tensor) -> RouterArgs:
        if logits.dim() != 2 or logits.dtype not in self.args:
            raise ValueError(f"{what}: logits [n_tok, n_expert] in fp32, fp16 or bf16")
        _expect(what, "logits", logits, (logits.shape[0], self.n_expert), logits.dtype, self.bias, rows=True)
        return self.args[logits.dtype]


def route(router: Router, logits: torch.Tensor, ids=None, wts=None, prow=None, counts=None, stream=None):
    """The picked experts' ids [n_tok, k] int32 (-1 where none is left) and weights [n_tok, k]; logits rows may lie apart.
    prow [n_tok, k] int32, if given: moe_combine's rows in entry order.  counts [n_expert] int32, if given: the tokens of
    each expert are added."""
    a = router.args_for("route", logits)
    shape = (logits.shape[0], router.k)
    if ids is None:
        ids = torch.empty(shape, dtype=torch.int32, device=logits.device)
    if wts is None:
        wts = torch.empty(shape, dtype=torch.float32, device=logits.device)
    _expect("route", "ids", ids, shape, torch.int32, logits)
    _expect("route", "wts", wts, shape, torch.float32, logits)
    _expect("route", "prow", prow, shape, torch.int32, logits)
    _expect("route", "counts", counts, (router.n_expert,), torch.int32, logits)
    _launch("route", lib().tsx_moe_route, logits, stream, C.byref(a), _p(logits), _ld(logits), _p(ids), _p(wts), _p(prow),
            _p(counts), shape[0])
    return ids, wts


def route_backward(router: Router, logits: torch.Tensor, ids: torch.Tensor, dwts: torch.Tensor, dlogits=None,
                   stream=None) -> torch.Tensor:
    """The weights' gradient dwts [n_tok, k] of the picks ids -> the logits' [n_tok, n_expert], in the logits' type."""
    a = router.args_for("route_backward", logits)
    shape = (logits.shape[0], router.k)
    if dlogits is None:
        dlogits = torch.empty(tuple(logits.shape), dtype=logits.dtype, device=logits.device)
    _expect("route_backward", "ids", ids, shape, torch.int32, logits)
    _expect("route_backward", "dwts", dwts, shape, torch.float32, logits)
    _expect("route_backward", "dlogits", dlogits, logits.shape, logits.dtype, logits, rows=True)
    _launch("route_backward", lib().tsx_moe_route_backward, logits, stream, C.byref(a), _p(logits), _ld(logits), _p(ids),
            _p(dwts), _p(dlogits), _ld(dlogits), shape[0])
    return dlogits


def group_entries(ids: torch.Tensor, k: int, n_expert: int, blobs_ptr: int, stride: int, bufs=None, stream=None):
    """Decode grouping (k_group): returns grp_ptr, grp_start, n_groups, ent_dst, ent_tok (device tensors)."""
    n_ent = ids.numel()
    cap = min(n_ent, n_expert)
    dev = ids.device
    if bufs is None:
        bufs = (torch.empty(cap, dtype=torch.int64, device=dev), torch.empty(cap + 1, dtype=torch.int32, device=dev),
                torch.empty(1, dtype=torch.int32, device=dev), torch.empty(n_ent, dtype=torch.int32, device=dev),
                torch.empty(n_ent, dtype=torch.int32, device=dev))
    gp, gs, ng, ed, et = bufs
    check(lib().tsx_moe_group(_p(ids), n_ent, k, n_expert, blobs_ptr, stride, _p(gp), _p(gs), _p(ng), _p(ed), _p(et),
                              _stream(stream)), "group_entries")
    return bufs


def group_resident(ids: torch.Tensor, k: int, n_expert: int, slot_of: torch.Tensor, slots_ptr: int, stride: int,
                   bufs, stream=None):
    """Decode grouping of a hybrid layer (k_group_hy): only entries whose expert has a slot; group blobs in slots."""
    gp, gs, ng, ed, et = bufs
    check(lib().tsx_moe_group_resident(_p(ids), ids.numel(), k, n_expert, _p(slot_of), slots_ptr, stride, _p(gp),
                                       _p(gs), _p(ng), _p(ed), _p(et), _stream(stream)), "group_resident")
    return bufs


def merge_rows(parts: torch.Tensor, rows: torch.Tensor, miss: torch.Tensor, stream=None) -> None:
    """parts[e] = rows[miss[e]] where miss[e] >= 0 (k_merge_cpu, compact rows)."""
    n_ent, n = parts.shape
    check(lib().tsx_moe_merge_rows(_p(parts), _p(rows), _p(miss), n_ent, n, _stream(stream)), "merge_rows")


def route_sort(ids: torch.Tensor, k: int, n_expert: int, bufs=None, stream=None):
    """The prompt's expert sort: bounds [E+1], ent_dst, ent_tok, rinv [n_ent], max_rows [1]."""
    n_ent = ids.numel()
    dev = ids.device
    if bufs is None:
        bufs = (torch.empty(n_expert + 1, dtype=torch.int32, device=dev), torch.empty(n_ent, dtype=torch.int32, device=dev),
                torch.empty(n_ent, dtype=torch.int32, device=dev), torch.empty(n_ent, dtype=torch.int32, device=dev),
                torch.empty(1, dtype=torch.int32, device=dev))
    b, ed, et, ri, mr = bufs
    check(lib().tsx_moe_route_sort(_p(ids), n_ent, k, n_expert, _p(b), _p(ed), _p(et), _p(ri), _p(mr), _stream(stream)),
          "route_sort")
    return bufs


def moe_combine(x, parts, wts, k: int, prow=None, shared=None, sgate=None, sg_stride: int = 1, stream=None) -> None:
    """x[t] += sum_j w[t][j] parts[p(t,j)] (+ sigmoid(sgate[t]) shared[t]), in place; a prow below 0 adds nothing."""
    n_tok, n = x.shape
    check(lib().tsx_moe_combine(_p(x), _p(parts), _p(prow), _p(wts), k, _p(shared), _p(sgate), sg_stride, n, n_tok,
                                _stream(stream)), "moe_combine")


def moe_combine_norm(x, parts, wts, k: int, norm_w, eps: float, h, hq=None, prow=None, shared=None, sgate=None,
                     sg_stride: int = 1, stream=None) -> None:
    """moe_combine, then h = rms(x) * norm_w and (hq given) its Q8_1 image: the MoE block's end (k_moe_out)."""
    n_tok, n = x.shape
    check(lib().tsx_moe_combine_norm(_p(x), _p(parts), _p(prow), _p(wts), k, _p(shared), _p(sgate), sg_stride, n, n_tok,
                                     _p(norm_w), eps, _p(h), _p(hq), _stream(stream)), "moe_combine_norm")


def moe_combine_backward(dy, parts, wts, k: int, prow=None, shared=None, sgate=None, sg_stride: int = 1, dwts=None,
                         dparts=None, dshared=None, dsgate=None, stream=None) -> None:
    """The gradients of moe_combine from dy [n_tok, n], into those of dwts [n_tok, k], dparts (parts' shape), dshared
    [n_tok, n] and dsgate [n_tok] that are given."""
    what = "moe_combine_backward"
    _expect(what, "dy", dy, (dy.shape[0], dy.shape[-1]), torch.float32)
    n_tok, n = dy.shape
    _expect(what, "parts", parts, (parts.shape[0], n), torch.float32, dy)
    if prow is None and parts.shape[0] < n_tok * k:
        raise ValueError(f"{what}: {parts.shape[0]} part rows for {n_tok} tokens x {k}")
    _expect(what, "wts", wts, (n_tok, k), torch.float32, dy)
    if prow is not None:
        _expect(what, "prow", prow.view(-1), (n_tok * k,), torch.int32, dy)
    _expect(what, "shared", shared, (n_tok, n), torch.float32, dy)
    if sgate is not None:
        left = sgate.untyped_storage().nbytes() // 4 - sgate.storage_offset()
        if sgate.dtype != torch.float32 or sgate.device != dy.device or sg_stride < 0 or (
                n_tok and left <= (n_tok - 1) * sg_stride):
            raise ValueError(f"{what}: sgate in fp32 on {dy.device}, a value per token {sg_stride} apart")
    _expect(what, "dwts", dwts, (n_tok, k), torch.float32, dy)
    _expect(what, "dparts", dparts, parts.shape, torch.float32, dy)
    _expect(what, "dshared", dshared, (n_tok, n), torch.float32, dy)
    _expect(what, "dsgate", dsgate, (n_tok,), torch.float32, dy)
    _launch(what, lib().tsx_moe_combine_backward, dy, stream, _p(dy), _p(parts), _p(prow), _p(wts), k, _p(shared),
            _p(sgate), sg_stride, n, n_tok, _p(dwts), _p(dparts), _p(dshared), _p(dsgate))


# ------------------------------------------------------------------ prefill
def mmq_q8_bytes(rows: int, cols: int) -> int:
    return lib().tsx_moe_mmq_q8_bytes(rows, cols)


def mmq_quantize(x, ids, ggml_type: int, cols: int, ld: int, rows: int, xq=None, stream=None) -> torch.Tensor:
    if xq is None:
        xq = torch.empty(mmq_q8_bytes(rows, cols), dtype=torch.uint8, device=x.device)
    check(lib().tsx_moe_mmq_quantize(_p(x), _p(ids), _p(xq), ggml_type, cols, ld, rows, _stream(stream)), "mmq_quantize")
    return xq


def mmq_quantize_route(x, ggml_type: int, logits, k: int, xq=None, ids=None, wts=None, stream=None):
    """mmq_quantize of the token rows of x (ids None) and native_router_topk of logits in one launch; returns
    (xq, ids, wts)."""
    rows, cols = x.shape
    n_expert = logits.shape[1]
    if xq is None:
        xq = torch.empty(mmq_q8_bytes(rows, cols), dtype=torch.uint8, device=x.device)
    if ids is None:
        ids = torch.empty((rows, k), dtype=torch.int32, device=x.device)
    if wts is None:
        wts = torch.empty((rows, k), dtype=torch.float32, device=x.device)
    check(lib().tsx_moe_mmq_quantize_route(_p(x), _p(xq), ggml_type, cols, x.stride(0), rows, _p(logits), _p(ids),
                                           _p(wts), n_expert, k, _stream(stream)), "mmq_quantize_route")
    return xq, ids, wts


def mmq_run(w, ggml_type: int, w_rows: int, w_cols: int, expert_bytes: int, n: int, xq, bounds, ids, total_rows: int,
            dst, ld_dst: int, max_rows: int = 0, stream=None) -> None:
    p = MmqProduct(w=_p(w), type=ggml_type, n=n, w_rows=w_rows, w_cols=w_cols, expert_bytes=expert_bytes, xq=_p(xq),
                   bounds=_p(bounds), ids=_p(ids), total_rows=total_rows, max_rows=max_rows, dst=_p(dst), ld_dst=ld_dst)
    check(lib().tsx_moe_mmq_run(C.byref(p), _stream(stream)), "mmq_run")


def mmq_swiglu(gu, rows: int, n_ff: int, interleaved: bool = False, h=None, stream=None) -> torch.Tensor:
    if h is None:
        h = torch.empty((rows, n_ff), dtype=torch.float32, device=gu.device)
    check(lib().tsx_moe_mmq_swiglu(_p(gu), _p(h), rows, n_ff, int(interleaved), _stream(stream)), "mmq_swiglu")
    return h


def mmq_gate_up_swiglu(w, ggml_type: int, n_ff: int, n_embd: int, expert_bytes: int, n: int, xq, x_rows: int, xids,
                       bounds, n_rows: int, hq=None, stream=None) -> torch.Tensor:
    """h = silu(x . gate) * (x . up) of every expert's sorted rows (x rows through xids), quantized into Q8_1 planes
    of n_rows rows and n_ff columns (the layout mmq_quantize writes)."""
    if hq is None:
        hq = torch.empty(mmq_q8_bytes(n_rows, n_ff), dtype=torch.uint8, device=w.device)
    check(lib().tsx_moe_mmq_gate_up_swiglu(_p(w), ggml_type, n_ff, n_embd, expert_bytes, n, _p(xq), x_rows, _p(xids),
                                            _p(bounds), n_rows, _p(hq), _stream(stream)), "mmq_gate_up_swiglu")
    return hq


# ------------------------------------------------------------------ adapters
class Adapters:
    """Low-rank adapters beside one projection (tsx_adapters): a [n, rank, n_in] and b [n, n_out, rank] in fp32, fp16 or
    bf16, each adapter's matrix dense; scale [n] fp32 or None (1).  Read at every call: they may be updated in place."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor | None = None):
        if a.dim() != 3 or b.dim() != 3 or a.dtype not in PLAIN_TYPES:
            raise ValueError("Adapters: a [n, rank, n_in] and b [n, n_out, rank] in fp32, fp16 or bf16")
        n, rank, n_in = a.shape
        n_out = b.shape[1]
        for name, t, rows, cols in (("a", a, rank, n_in), ("b", b, n_out, rank)):
            if tuple(t.shape) != (n, rows, cols) or t.dtype != a.dtype or t.device != a.device:
                raise ValueError(f"Adapters: {name} is {t.dtype} {tuple(t.shape)} on {t.device}, not {a.dtype} "
                                 f"{(n, rows, cols)} on {a.device}")
            if t.numel() and not t[0].is_contiguous():
                raise ValueError(f"Adapters: {name}'s matrices are not dense (strides {t.stride()})")
        _expect("Adapters", "scale", scale, (n,), torch.float32, a)
        self.a, self.b, self.scale = a, b, scale
        self.n, self.rank, self.n_in, self.n_out = n, rank, n_in, n_out
        self.args = AdapterArgs(type=PLAIN_TYPES[a.dtype], n=n, rank=rank, n_in=n_in, n_out=n_out, a=a.data_ptr(),
                                b=b.data_ptr(), a_stride=a.stride(0) if n > 1 else rank * n_in,
                                b_stride=b.stride(0) if n > 1 else rank * n_out,
                                scale=None if scale is None else scale.data_ptr())


def adapters(ad: Adapters, ids: torch.Tensor, x: torch.Tensor, y: torch.Tensor, base: torch.Tensor | None = None,
             stream=None) -> torch.Tensor:
    """y[j] = base[j] + scale B (A x[j]) with the adapter ids[j] (int32; outside [0, n): none), rows of x [rows, n_in],
    base and y [rows, n_out] possibly apart; base may be y, or None for 0."""
    rows = ids.shape[0]
    _expect("adapters", "ids", ids, (rows,), torch.int32, x)
    _expect("adapters", "x", x, (rows, ad.n_in), torch.float32, ad.a, rows=True)
    _expect("adapters", "y", y, (rows, ad.n_out), torch.float32, x, rows=True)
    _expect("adapters", "base", base, (rows, ad.n_out), torch.float32, x, rows=True)
    _launch("adapters", lib().tsx_moe_adapters, x, stream, C.byref(ad.args), _p(ids), _p(x), _ld(x), _p(base), _ld(base),
            _p(y), _ld(y), rows)
    return y


def adapters_scratch_bytes(ad: Adapters, rows: int) -> int:
    return lib().tsx_moe_adapters_scratch_bytes(C.byref(ad.args), rows)


def adapters_backward(ad: Adapters, ids: torch.Tensor, x: torch.Tensor, dy: torch.Tensor, dx=None, da=None, db=None,
                      dbase=None, scratch=None, stream=None) -> None:
    """The gradients of adapters() from dy [rows, n_out], into those of dx [rows, n_in] (= dbase + ..), da [n, rank, n_in]
    and db [n, n_out, rank] (fp32) that are given."""
    what, rows = "adapters_backward", ids.shape[0]
    _expect(what, "ids", ids, (rows,), torch.int32, x)
    _expect(what, "x", x, (rows, ad.n_in), torch.float32, ad.a, rows=True)
    _expect(what, "dy", dy, (rows, ad.n_out), torch.float32, x, rows=True)
    _expect(what, "dx", dx, (rows, ad.n_in), torch.float32, x, rows=True)
    _expect(what, "dbase", dbase, (rows, ad.n_in), torch.float32, x, rows=True)
    _expect(what, "da", da, ad.a.shape, torch.float32, x)
    _expect(what, "db", db, ad.b.shape, torch.float32, x)
    need = adapters_scratch_bytes(ad, rows)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
        if stream is not None:
            scratch.record_stream(stream)  # its memory goes back to the current stream's allocations when this returns
    elif scratch.device != x.device or not scratch.is_contiguous() or scratch.numel() * scratch.element_size() < need:
        raise ValueError(f"{what}: scratch of {need} bytes on {x.device} (adapters_scratch_bytes)")
    _launch(what, lib().tsx_moe_adapters_backward, x, stream, C.byref(ad.args), _p(ids), _p(x), _ld(x), _p(dy), _ld(dy),
            _p(dbase), _ld(dbase), _p(dx), _ld(dx), _p(da), _p(db), rows, _p(scratch))


# ------------------------------------------------------------------ checks and data
def subblock_sums(ggml_type: int, w, n_in: int, n_rows: int, x_q8_1, ncols: int, stream=None):
    nsub = n_in // 32
    sums = torch.empty((n_rows, ncols, nsub), dtype=torch.int32, device=w.device)
    qsums = torch.empty((n_rows, ncols, nsub), dtype=torch.int32, device=w.device)
    check(lib().tsx_moe_subblock_sums(ggml_type, _p(w), n_in, n_rows, _p(x_q8_1), ncols, _p(sums), _p(qsums),
                                      _stream(stream)), "subblock_sums")
    return sums, qsums


def quantize_weights(ggml_type: int, x: np.ndarray) -> np.ndarray:
    """Host: float32 [rows, cols] -> GGUF blocks uint8 [rows, row_bytes]."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    rows, cols = x.shape
    rb = iq_row_bytes(ggml_type, cols)
    out = np.empty((rows, rb), dtype=np.uint8)
    check(lib().tsx_moe_quantize_weights(ggml_type, x.ctypes.data, rows, cols, out.ctypes.data), "quantize_weights")
    return out
