"""The NVFP4 linear with its epilogue (``Runtime.linear_fused``) and its form
for rows sorted by group (``Runtime.linear_grouped``): argument checks and the
call. Weights-only NVFP4 on 16-bit or FP32 activations, for inference; the lab's
linear has FP32 activations and leaves bias and activation to its caller
(vllm_nvfp4_opencl/linear.py:49-70).
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .experts import TYPES, _row_stride, _rows_of, on_stream, refuse_tangents, stream_of, written
from .runtime import ACTIVATIONS

# A call on one token is over on the GPU in a few microseconds, less than its way through Python: messages are made only
# when they are raised, and nothing is asked of a tensor twice.


# The library's limit, checked here because ctypes would pass a larger number's low 32 bits.
MAX_ROWS = 1 << 30


def _refuse(message):
    raise ValueError(message)


def _check(matrix, x, bias, activation, others):
    """Outputs a row, after the checks that both forms share; ``others``: the optional tensors besides bias."""
    if not (x.is_cuda and x.dtype in TYPES and x.dim() >= 1 and x.shape[-1] == matrix.cols):
        _refuse("x must be a CUDA bfloat16, float16 or float32 tensor [..., cols]")
    if x.numel() > MAX_ROWS * matrix.cols:
        _refuse("x must have at most 2^30 rows")
    device, home = x.device, matrix.device
    if home is not None and device.index != home:
        _refuse(f"x is on {device} but the matrix is resident on cuda:{home}")
    recorded = x.requires_grad
    for t in others:
        if t is not None:
            if t.device != device:
                _refuse("bias, offsets, residual and out must be on x's device")
            recorded = recorded or t.requires_grad
    if bias is not None:
        if bias.device != device:
            _refuse("bias, offsets, residual and out must be on x's device")
        if bias.dtype not in TYPES or (bias.shape != (matrix.groups, matrix.rows) and
                                       (matrix.groups != 1 or bias.shape != (matrix.rows,))):
            _refuse("bias must be bfloat16, float16 or float32, [rows] or [groups, rows] of the matrix")
        recorded = recorded or bias.requires_grad
    if recorded and torch.is_grad_enabled():
        _refuse("the NVFP4 linear records no gradient: call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0:
        refuse_tangents((x, bias, *others))
    if activation is None:
        return matrix.rows
    if activation not in ACTIVATIONS:
        _refuse(f"unknown activation {activation!r}")
    if not activation.endswith("_mul"):
        return matrix.rows
    if matrix.rows % 2:
        _refuse("a gated activation needs an even number of weight rows")
    return matrix.rows // 2


def _workspace(rt, matrix, x, at, stride, grouped):
    """(tensor, address, bytes) of the call's device workspace, from torch's allocator on the current stream. The
    tensor is held until the kernels are enqueued; its memory then goes to later work of the same stream."""
    if at % 16 == 0 and stride % 8 == 0 and stride >= matrix.cols and x.dtype != torch.float32:
        return None, None, 0  # rows that every kernel reads where they lie
    size = rt.lib.nvfp4_linear_workspace_bytes(matrix.handle, at, TYPES[x.dtype], stride, x.shape[0], grouped)
    if not size:
        return None, None, 0
    held = torch.empty(size, dtype=torch.uint8, device=x.device)
    return held, held.data_ptr(), size


def _rows2d(t, cols):
    return _rows_of(t if t.dim() == 2 else t.reshape(-1, cols))


def _bias(bias):
    """(bias, address, type): the tensor is held until the kernels are enqueued."""
    if bias is None:
        return None, None, 0
    bias = bias.contiguous()
    return bias, bias.data_ptr(), TYPES[bias.dtype]


def _linear(rt, matrix, x, bias, activation, residual, out, width, shape):
    x2 = _rows2d(x, matrix.cols)
    y = x.new_empty(shape) if out is None else out
    stride = width
    if out is not None:
        try:
            y2 = out if out.dim() == 2 else out.view(-1, width)
        except RuntimeError:
            y2 = None
        if y2 is None or (y2.stride(1) != 1 and width != 1) or (y2.shape[0] > 1 and y2.stride(0) < width):
            _refuse("out must have contiguous columns and even rows")
        stride = _row_stride(y2)
    count = x2.shape[0]
    if count == 0:
        return y
    r2, r_at, r_stride = None, None, 0
    if residual is not None:
        r2 = _rows2d(residual, width)
        r_at, r_stride = r2.data_ptr(), _row_stride(r2)
    _held_bias, b_at, b_type = _bias(bias)
    x_at, x_stride = x2.data_ptr(), _row_stride(x2)
    _held, space, size = _workspace(rt, matrix, x2, x_at, x_stride, 0)
    rt._check(
        rt.lib.nvfp4_linear_fused(rt.handle, matrix.handle, x_at, TYPES[x.dtype], x_stride, count, b_at, b_type,
                                  ACTIVATIONS[activation], r_at, r_stride, y.data_ptr(), stride, space, size,
                                  stream_of(x.device)),
        "nvfp4_linear_fused")
    return y if out is None else written(y)


def linear_fused(rt, matrix, x, bias, activation, residual, out, stream):
    width = _check(matrix, x, bias, activation, (residual, out))
    if matrix.groups != 1:
        _refuse("a matrix of several groups runs through linear_grouped")
    shape = (*x.shape[:-1], width)
    for t in (residual, out):
        if t is not None and (t.shape != shape or t.dtype != x.dtype):
            _refuse(f"residual and out must be of x's type, [..., {width}]")
    if stream is None:
        return _linear(rt, matrix, x, bias, activation, residual, out, width, shape)
    return on_stream(stream, (x, bias, residual, out),
                     lambda: _linear(rt, matrix, x, bias, activation, residual, out, width, shape))


def _grouped(rt, matrix, x, offsets, bias, activation, out, shape):
    y = out if out is not None else x.new_empty(shape)
    count, width = shape
    if count == 0:
        return y
    x2, o = _rows_of(x), offsets.contiguous()
    _held_bias, b_at, b_type = _bias(bias)
    x_at, x_stride = x2.data_ptr(), _row_stride(x2)
    _held, space, size = _workspace(rt, matrix, x2, x_at, x_stride, 1)
    rt._check(
        rt.lib.nvfp4_linear_grouped(rt.handle, matrix.handle, x_at, TYPES[x.dtype], x_stride, count, o.data_ptr(),
                                    b_at, b_type, ACTIVATIONS[activation], y.data_ptr(),
                                    width if out is None else _row_stride(y), 1 if out is None else 0, space, size,
                                    stream_of(x.device)),
        "nvfp4_linear_grouped")
    return y if out is None else written(y)


def linear_grouped(rt, matrix, x, offsets, bias, activation, out, stream):
    width = _check(matrix, x, bias, activation, (offsets, out))
    if x.dim() != 2:
        _refuse("x must be [rows, cols]")
    if offsets.dtype != torch.int32 or offsets.shape != (matrix.groups + 1,):
        _refuse("offsets must be int32 [groups + 1]")
    shape = (x.shape[0], width)
    if out is not None and (out.shape != shape or out.dtype != x.dtype or (out.stride(1) != 1 and width != 1)
                            or (shape[0] > 1 and out.stride(0) < width)):
        _refuse(f"out must be of x's type, [rows, {width}] with contiguous columns")
    if stream is None:
        return _grouped(rt, matrix, x, offsets, bias, activation, out, shape)
    return on_stream(stream, (x, offsets, bias, out),
                     lambda: _grouped(rt, matrix, x, offsets, bias, activation, out, shape))


__all__ = ["linear_fused", "linear_grouped"]
