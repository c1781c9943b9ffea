"""Token rows sorted by expert and brought back, with their gradients.

The pieces between a router and experts that are not a ``MoeBank`` (other
products, other top-k, training): ``expert_sort`` copies every token's row to
its experts' places in expert order, the caller runs the experts on the rows
(``Runtime.linear_grouped`` for NVFP4 weights, with ``order.offsets``), and
``expert_return`` weights and sums every token's rows. Both are differentiable
(once): the sort in x, the return in the rows, the weights and the residual.
They are reached as ``Runtime.expert_sort`` and ``Runtime.expert_return``; the
lab has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from .runtime import CUDA_STREAM_LEGACY

# Element types of the C ABI (NVFP4_TYPE_*).
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_TOPK, MAX_EXPERTS = 64, 1024
# Checked here although the library does so too: its arguments are 32-bit, and ctypes would pass a larger number's low bits.
MAX_PICKS, MAX_HIDDEN = 2 ** 31 - 16386, 1 << 24


class ExpertOrder(NamedTuple):
    """Where ``expert_sort`` put the picks (int32 CUDA tensors). A pick may be
    dropped after the sort too (a capacity limit), by an ``inverse`` of its own
    with -1 there: ``order._replace(inverse=...)``. The return leaves it out,
    and the gradient of its row is zero. No two picks may name the same row."""

    perm: torch.Tensor     # [T*K] flat pick token*K + k of each row, -1 past the last expert's rows
    inverse: torch.Tensor  # [T, K] row of each pick, -1 where its id names no expert
    offsets: torch.Tensor  # [experts + 1] first row of each expert, then the number of rows in use
    experts: int


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous columns (a row stride is kept)."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def refuse_tangents(tensors):
    """Raises where one of the tensors (or None) carries a forward-mode derivative: ``requires_grad`` does not say so, and
    the result would come without it. Asked only within a dual level (``forward_ad._current_level``): there are none
    outside."""
    if not torch._C._is_fwd_grad_enabled():
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("no forward-mode derivative goes through this operator: call it on the primal tensors "
                             "(torch.autograd.forward_ad.unpack_dual)")


def on_stream(stream, tensors, call):
    """``call()`` on ``stream``, of the GPU of the first tensor: what it allocates then belongs to that stream, and the
    given tensors are kept from reuse until the stream is done with them."""
    if stream.device != tensors[0].device:
        raise ValueError(f"the stream is of {stream.device}, the tensors are on {tensors[0].device}")
    with torch.cuda.stream(stream):
        result = call()
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return result


def written(out):
    """Tells autograd that a call has written to a tensor of the caller's: one that it keeps for a gradient must not change
    without a word."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return out


def stream_of(device) -> int:
    """torch's current stream on ``device`` as the C ABI takes it (its default stream has handle 0, which the ABI would
    read as the runtime's own)."""
    return torch._C._cuda_getCurrentRawStream(device.index) or CUDA_STREAM_LEGACY


# ------------------------------------------------------------------ one call each


def _sort(rt, x, ids, experts):
    tokens, hidden = x.shape
    topk = ids.shape[1]
    picks = tokens * topk
    rows = x.new_empty((picks, hidden))
    table = torch.empty(2 * picks + experts + 1, dtype=torch.int32, device=x.device)
    perm, inverse, offsets = table.split((picks, picks, experts + 1))
    inverse = inverse.view(tokens, topk)
    if tokens == 0:
        offsets.zero_()
        return rows, perm, inverse, offsets
    x, ids = _rows_of(x), _rows_of(ids)
    rt._check(
        rt.lib.nvfp4_expert_sort(
            rt.handle, x.data_ptr(), TYPES[x.dtype], _row_stride(x), tokens, hidden, ids.data_ptr(),
            ids.element_size(), _row_stride(ids), topk, experts, rows.data_ptr(), perm.data_ptr(),
            inverse.data_ptr(), offsets.data_ptr(), stream_of(x.device)),
        "nvfp4_expert_sort")
    return rows, perm, inverse, offsets


def _return(rt, rows, inverse, weights, residual, out):
    tokens, topk = inverse.shape
    hidden = rows.shape[1]
    given = out is not None
    if not given:
        out = rows.new_empty((tokens, hidden))
    if tokens == 0:
        return out
    rows = _rows_of(rows)
    if residual is not None:
        residual = _rows_of(residual)
    if weights is not None:
        weights = weights.contiguous()
    rt._check(
        rt.lib.nvfp4_expert_return(
            rt.handle, rows.data_ptr(), TYPES[rows.dtype], _row_stride(rows), inverse.data_ptr(),
            weights.data_ptr() if weights is not None else None,
            TYPES[weights.dtype] if weights is not None else 0,
            residual.data_ptr() if residual is not None else None,
            _row_stride(residual) if residual is not None else 0, tokens, topk, hidden, out.data_ptr(),
            _row_stride(out), stream_of(rows.device)),
        "nvfp4_expert_return")
    return written(out) if given else out


def _return_backward(rt, dout, rows, inverse, offsets, weights, experts, need_rows, need_weights):
    tokens, topk = inverse.shape
    hidden = dout.shape[1]
    drows = dout.new_empty((tokens * topk, hidden)) if need_rows else None
    dweights = torch.empty((tokens, topk), dtype=weights.dtype, device=dout.device) if need_weights else None
    if tokens == 0:
        return drows, dweights
    dout = _rows_of(dout)
    if rows is not None:
        rows = _rows_of(rows)
    if weights is not None:
        weights = weights.contiguous()
    rt._check(
        rt.lib.nvfp4_expert_return_backward(
            rt.handle, dout.data_ptr(), TYPES[dout.dtype], _row_stride(dout),
            rows.data_ptr() if need_weights else None, _row_stride(rows) if need_weights else 0,
            inverse.data_ptr(), offsets.data_ptr(), weights.data_ptr() if weights is not None else None,
            TYPES[weights.dtype] if weights is not None else 0, tokens, topk, hidden, experts,
            drows.data_ptr() if need_rows else None, dweights.data_ptr() if need_weights else None,
            stream_of(dout.device)),
        "nvfp4_expert_return_backward")
    return drows, dweights


# ------------------------------------------------------------------ gradients


# Of a gradient there is no gradient: where one is recorded (create_graph) the result says so when it is asked for. The
# guard costs several microseconds of the host, which an ordinary backward pass goes without.


def _sort_gradient(ctx, drows):
    if forward_ad._current_level >= 0:
        refuse_tangents((drows,))
    (inverse,) = ctx.saved_tensors
    return _return(ctx.rt, drows, inverse, None, None, None), None, None, None, None


def _return_gradient(ctx, dout):
    if forward_ad._current_level >= 0:
        refuse_tangents((dout,))
    rows, weights, inverse, offsets = ctx.saved_tensors
    need_rows, need_weights, need_residual = ctx.needs_input_grad[:3]
    drows = dweights = None
    if need_rows or need_weights:
        drows, dweights = _return_backward(ctx.rt, dout, rows, inverse, offsets, weights, ctx.experts, need_rows,
                                           need_weights)
    return drows, dweights, dout if need_residual else None, None, None


_sort_gradient_once = torch.autograd.function.once_differentiable(_sort_gradient)
_return_gradient_once = torch.autograd.function.once_differentiable(_return_gradient)


class _ExpertSort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rt, ids, experts, record):
        # The order goes out by the record: numbers without a gradient, which autograd need not see.
        rows, *order = _sort(rt, x, ids, experts)
        record.extend(order)
        ctx.rt = rt
        ctx.save_for_backward(order[1])
        return rows

    @staticmethod
    def backward(ctx, drows):
        return _sort_gradient_once(ctx, drows) if torch.is_grad_enabled() else _sort_gradient(ctx, drows)


class _ExpertReturn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, residual, rt, order):
        ctx.rt = rt
        ctx.experts = order.experts
        # The rows are kept only for the weights' gradient.
        keep = weights is not None and ctx.needs_input_grad[1]
        ctx.save_for_backward(rows if keep else None, weights, order.inverse, order.offsets)
        return _return(rt, rows, order.inverse, weights, residual, None)

    @staticmethod
    def backward(ctx, dout):
        return _return_gradient_once(ctx, dout) if torch.is_grad_enabled() else _return_gradient(ctx, dout)


# ------------------------------------------------------------------ checks


def _require(condition, message):
    if not condition:
        raise ValueError(message)


def expert_sort(rt, x, ids, experts: int, stream=None):
    _require(x.is_cuda and x.dim() == 2 and x.dtype in TYPES and x.shape[1] > 0,
             "x must be a CUDA bfloat16, float16 or float32 tensor [tokens, hidden]")
    _require(ids.dtype in (torch.int32, torch.int64) and ids.dim() == 2 and ids.shape[0] == x.shape[0]
             and ids.device == x.device, "ids must be int32 or int64 [tokens, topk] on x's device")
    _require(1 <= ids.shape[1] <= MAX_TOPK, "the expert sort supports 1 to 64 picks a token")
    _require(ids.numel() <= MAX_PICKS and x.shape[1] <= MAX_HIDDEN,
             "the expert sort supports at most 2^31 - 16386 picks and 2^24 columns")
    experts = int(experts)
    _require(1 <= experts <= MAX_EXPERTS, "the expert sort supports 1 to 1024 experts")
    if forward_ad._current_level >= 0:
        refuse_tangents((x,))
    grad = x.requires_grad and torch.is_grad_enabled()

    def call():
        if grad:
            record = []
            return _ExpertSort.apply(x, rt, ids, experts, record), *record
        return _sort(rt, x, ids, experts)

    rows, perm, inverse, offsets = call() if stream is None else on_stream(stream, (x, ids), call)
    return rows, ExpertOrder(perm, inverse, offsets, experts)


def expert_return(rt, rows, order: ExpertOrder, weights=None, residual=None, out=None, stream=None):
    inverse, offsets = order.inverse, order.offsets
    _require(inverse.dtype == torch.int32 and offsets.dtype == torch.int32 and inverse.dim() == 2
             and inverse.is_contiguous() and offsets.is_contiguous() and offsets.numel() == order.experts + 1
             and offsets.device == inverse.device,
             "order must come from expert_sort: contiguous int32 inverse [tokens, topk] and offsets [experts + 1]")
    tokens, topk = inverse.shape
    device, hidden = rows.device, rows.shape[-1]
    _require(rows.is_cuda and rows.dim() == 2 and rows.dtype in TYPES and rows.shape[0] == tokens * topk and hidden > 0
             and device == inverse.device,
             "rows must be a CUDA bfloat16, float16 or float32 tensor [tokens * topk, hidden] on the order's device")
    _require(rows.shape[0] <= MAX_PICKS and hidden <= MAX_HIDDEN,
             "the expert return supports at most 2^31 - 16386 rows and 2^24 columns")
    grad = rows.requires_grad
    if weights is not None:
        _require(weights.shape == inverse.shape and weights.dtype in TYPES and weights.device == device,
                 "weights must be bfloat16, float16 or float32 [tokens, topk] on the rows' device")
        grad = grad or weights.requires_grad
    if residual is not None:
        _require(residual.shape == (tokens, hidden) and residual.dtype == rows.dtype and residual.device == device,
                 "residual must match the rows' type and device, [tokens, hidden]")
        grad = grad or residual.requires_grad
    grad = grad and torch.is_grad_enabled()
    if forward_ad._current_level >= 0:
        refuse_tangents((rows, weights, residual))
    if out is not None:
        _require(out.shape == (tokens, hidden) and out.dtype == rows.dtype and out.device == device
                 and (out.stride(1) == 1 or hidden == 1) and (tokens < 2 or out.stride(0) >= hidden),
                 "out must match the rows' type and device, [tokens, hidden] with contiguous columns")
        _require(not grad and not out.requires_grad, "out cannot be given where gradients are recorded")

    def call():
        if grad:
            return _ExpertReturn.apply(rows, weights, residual, rt, order)
        return _return(rt, rows, inverse, weights, residual, out)

    return call() if stream is None else on_stream(stream, (rows, inverse, offsets, weights, residual, out), call)


__all__ = ["ExpertOrder", "expert_return", "expert_sort"]
