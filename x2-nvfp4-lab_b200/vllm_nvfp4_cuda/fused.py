"""The NVFP4 linear with its epilogue (``Runtime.linear_fused``) and its form
for rows sorted by group (``Runtime.linear_grouped``): argument checks and the
call. Weights-only NVFP4 on 16-bit or FP32 activations, for inference; the lab's
linear has FP32 activations and leaves bias and activation to its caller
(vllm_nvfp4_opencl/linear.py:49-70).
"""

from __future__ import annotations

import torch

from .experts import TYPES, _row_stride, _rows_of, on_stream, stream_of
from .runtime import ACTIVATIONS


def _require(condition, message):
    if not condition:
        raise ValueError(message)


def _checks(matrix, x, bias, activation, tensors):
    _require(x.is_cuda and x.dtype in TYPES and x.dim() >= 1 and x.shape[-1] == matrix.cols,
             "x must be a CUDA bfloat16, float16 or float32 tensor [..., cols]")
    home = matrix.device
    _require(home is None or x.device.index == home,
             f"x is on {x.device} but the matrix is resident on cuda:{home}")
    for name, t in tensors:
        _require(t is None or t.device == x.device, f"{name} must be on x's device")
    _require(activation in ACTIVATIONS, f"unknown activation {activation!r}")
    _require(not activation or not activation.endswith("_mul") or matrix.rows % 2 == 0,
             "a gated activation needs an even number of weight rows")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for _, t in (("x", x), *tensors)):
        raise ValueError("the NVFP4 linear records no gradient: call it under torch.no_grad() or on detached tensors")
    shape = (matrix.rows,) if matrix.groups == 1 else (matrix.groups, matrix.rows)
    if bias is not None:
        _require(bias.dtype in TYPES and tuple(bias.shape) in (shape, (matrix.groups, matrix.rows)),
                 f"bias must be bfloat16, float16 or float32 {list(shape)}")
    return matrix.rows // 2 if activation and activation.endswith("_mul") else matrix.rows


def _workspace(rt, matrix, x, grouped):
    """(tensor, address, bytes) of the call's device workspace, from torch's allocator on the current stream. The
    tensor is held until the kernels are enqueued; its memory then goes to later work of the same stream."""
    size = rt.lib.nvfp4_linear_workspace_bytes(matrix.handle, x.data_ptr(), TYPES[x.dtype], _row_stride(x), x.shape[0],
                                               grouped)
    if not size:
        return None, None, 0
    held = torch.empty(size, dtype=torch.uint8, device=x.device)
    return held, held.data_ptr(), size


def linear_fused(rt, matrix, x, bias, activation, residual, out, stream):
    width = _checks(matrix, x, bias, activation, (("bias", bias), ("residual", residual), ("out", out)))
    _require(matrix.groups == 1, "a matrix of several groups runs through linear_grouped")
    shape = (*x.shape[:-1], width)
    for name, t in (("residual", residual), ("out", out)):
        _require(t is None or (tuple(t.shape) == shape and t.dtype == x.dtype),
                 f"{name} must be of x's type, [..., {width}]")

    def rows2d(t, cols):
        return _rows_of(t if t.dim() == 2 else t.reshape(-1, cols))

    def call():
        x2 = rows2d(x, matrix.cols)
        if out is None:
            y, stride = x.new_empty(shape), width
        else:
            y = out
            try:
                y2 = out if out.dim() == 2 else out.view(-1, width)
            except RuntimeError:
                y2 = None
            _require(y2 is not None and (y2.stride(1) == 1 or width == 1)
                     and (y2.shape[0] < 2 or y2.stride(0) >= width), "out must have contiguous columns and even rows")
            stride = _row_stride(y2)
        if x2.shape[0] == 0:
            return y
        r2 = rows2d(residual, width) if residual is not None else None
        b = bias.contiguous() if bias is not None else None
        _held, space, size = _workspace(rt, matrix, x2, 0)
        rt._check(
            rt.lib.nvfp4_linear_fused(
                rt.handle, matrix.handle, x2.data_ptr(), TYPES[x.dtype], _row_stride(x2), x2.shape[0],
                b.data_ptr() if b is not None else None, TYPES[b.dtype] if b is not None else 0,
                ACTIVATIONS[activation], r2.data_ptr() if r2 is not None else None,
                _row_stride(r2) if r2 is not None else 0, y.data_ptr(), stride, space, size,
                stream_of(x.device)),
            "nvfp4_linear_fused")
        return y

    return on_stream(stream, (x, bias, residual, out), call)


def linear_grouped(rt, matrix, x, offsets, bias, activation, out, stream):
    width = _checks(matrix, x, bias, activation, (("bias", bias), ("offsets", offsets), ("out", out)))
    _require(x.dim() == 2, "x must be [rows, cols]")
    _require(offsets.dtype == torch.int32 and tuple(offsets.shape) == (matrix.groups + 1,),
             "offsets must be int32 [groups + 1]")
    shape = (x.shape[0], width)
    if out is not None:
        _require(tuple(out.shape) == shape and out.dtype == x.dtype and (out.stride(1) == 1 or width == 1)
                 and (shape[0] < 2 or out.stride(0) >= width),
                 f"out must be of x's type, [rows, {width}] with contiguous columns")

    def call():
        y = out if out is not None else x.new_empty(shape)
        if shape[0] == 0:
            return y
        x2, o = _rows_of(x), offsets.contiguous()
        b = bias.contiguous() if bias is not None else None
        _held, space, size = _workspace(rt, matrix, x2, 1)
        rt._check(
            rt.lib.nvfp4_linear_grouped(
                rt.handle, matrix.handle, x2.data_ptr(), TYPES[x.dtype], _row_stride(x2), shape[0], o.data_ptr(),
                b.data_ptr() if b is not None else None, TYPES[b.dtype] if b is not None else 0,
                ACTIVATIONS[activation], y.data_ptr(), _row_stride(y), 1 if out is None else 0, space, size,
                stream_of(x.device)),
            "nvfp4_linear_grouped")
        return y

    return on_stream(stream, (x, offsets, bias, out), call)


__all__ = ["linear_fused", "linear_grouped"]
