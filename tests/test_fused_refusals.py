"""What the fused linears and the expert sort and return refuse, before anything reaches a GPU: tensors without memory
for the Python checks, the C entry points for theirs, and the overlap rule of their rows (no GPU)."""

from __future__ import annotations

import ctypes as C
from types import SimpleNamespace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from vllm_nvfp4_cuda import experts, fused
from vllm_nvfp4_cuda.runtime import load_library

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class _Unreached:
    """Stands for the runtime: a call that is refused in time never asks it for anything."""

    def __getattr__(self, name):
        raise AssertionError(f"the runtime was reached ({name})")


RT = _Unreached()


def _cuda(*shape, dtype=BF16, device="cuda:0"):
    return torch.empty(shape, dtype=dtype, device=device)


def _matrix(rows=64, cols=64, groups=1, device=0):
    return SimpleNamespace(rows=rows, cols=cols, groups=groups, device=device)


def _linear(m, x, bias=None, activation=None, residual=None, out=None):
    return fused.linear_fused(RT, m, x, bias, activation, residual, out, None)


def _grouped(m, x, offsets, bias=None, activation=None, out=None):
    return fused.linear_grouped(RT, m, x, offsets, bias, activation, out, None)


LINEAR = {
    "x on the CPU": lambda: _linear(_matrix(), _cuda(3, 64, device="cpu")),
    "x in 64 bits": lambda: _linear(_matrix(), _cuda(3, 64, dtype=torch.float64)),
    "x of other columns": lambda: _linear(_matrix(), _cuda(3, 48)),
    "x without axes": lambda: _linear(_matrix(), _cuda()),
    "x on another GPU": lambda: _linear(_matrix(), _cuda(3, 64, device="cuda:1")),
    "bias on another GPU": lambda: _linear(_matrix(), _cuda(3, 64), _cuda(64, device="cuda:1")),
    "bias of another length": lambda: _linear(_matrix(), _cuda(3, 64), _cuda(63)),
    "bias of integers": lambda: _linear(_matrix(), _cuda(3, 64), _cuda(64, dtype=torch.int32)),
    "unknown activation": lambda: _linear(_matrix(), _cuda(3, 64), activation="tanh"),
    "gate over odd rows": lambda: _linear(_matrix(65), _cuda(3, 64), activation="silu_mul"),
    "residual of another type": lambda: _linear(_matrix(), _cuda(3, 64), residual=_cuda(3, 64, dtype=F32)),
    "residual of the ungated width": lambda: _linear(_matrix(), _cuda(3, 64), activation="silu_mul",
                                                     residual=_cuda(3, 64)),
    "out of another shape": lambda: _linear(_matrix(), _cuda(3, 64), out=_cuda(4, 64)),
    "out without contiguous columns": lambda: _linear(_matrix(), _cuda(3, 64), out=_cuda(64, 3).t()),
    "out of one row repeated": lambda: _linear(_matrix(), _cuda(3, 64), out=_cuda(1, 64).expand(3, 64)),
    "out of uneven rows": lambda: _linear(_matrix(), _cuda(2, 2, 64), out=_cuda(2, 3, 64)[:, :2]),
    "x with a gradient": lambda: _linear(_matrix(), _cuda(3, 64).requires_grad_()),
    "bias with a gradient": lambda: _linear(_matrix(), _cuda(3, 64), _cuda(64).requires_grad_()),
    "matrix of several groups": lambda: _linear(_matrix(groups=2), _cuda(3, 64)),
    "rows with a leading axis": lambda: _grouped(_matrix(groups=2), _cuda(1, 3, 64), _cuda(3, dtype=torch.int32)),
    "offsets of 64 bits": lambda: _grouped(_matrix(groups=2), _cuda(3, 64), _cuda(3, dtype=torch.int64)),
    "offsets without an end": lambda: _grouped(_matrix(groups=2), _cuda(3, 64), _cuda(2, dtype=torch.int32)),
    "offsets on the CPU": lambda: _grouped(_matrix(groups=2), _cuda(3, 64),
                                           _cuda(3, dtype=torch.int32, device="cpu")),
    "one bias for all groups": lambda: _grouped(_matrix(groups=2), _cuda(3, 64), _cuda(3, dtype=torch.int32),
                                                _cuda(64)),
    "grouped out of another type": lambda: _grouped(_matrix(groups=2), _cuda(3, 64), _cuda(3, dtype=torch.int32),
                                                    out=_cuda(3, 64, dtype=F16)),
}


def _sort(x=None, ids=None, n=4):
    x = _cuda(5, 8) if x is None else x
    return experts.expert_sort(RT, x, _cuda(5, 2, dtype=torch.int32) if ids is None else ids, n)


def _order(tokens=5, topk=2, n=4, device="cuda:0", dtype=torch.int32):
    return experts.ExpertOrder(_cuda(tokens * topk, dtype=dtype, device=device),
                               _cuda(tokens, topk, dtype=dtype, device=device),
                               _cuda(n + 1, dtype=dtype, device=device), n)


def _return(rows=None, order=None, weights=None, residual=None, out=None):
    rows = _cuda(10, 8) if rows is None else rows
    return experts.expert_return(RT, rows, order or _order(), weights, residual, out)


EXPERTS = {
    "x on the CPU": lambda: _sort(_cuda(5, 8, device="cpu")),
    "x in 64 bits": lambda: _sort(_cuda(5, 8, dtype=torch.float64)),
    "x of one axis": lambda: _sort(_cuda(5)),
    "x without columns": lambda: _sort(_cuda(5, 0)),
    "ids of 16 bits": lambda: _sort(ids=_cuda(5, 2, dtype=torch.int16)),
    "ids of other tokens": lambda: _sort(ids=_cuda(4, 2, dtype=torch.int32)),
    "ids on another GPU": lambda: _sort(ids=_cuda(5, 2, dtype=torch.int32, device="cuda:1")),
    "no picks": lambda: _sort(ids=_cuda(5, 0, dtype=torch.int32)),
    "65 picks": lambda: _sort(ids=_cuda(5, 65, dtype=torch.int32)),
    "no experts": lambda: _sort(n=0),
    "1025 experts": lambda: _sort(n=1025),
    "rows of other tokens": lambda: _return(_cuda(9, 8)),
    "rows in 64 bits": lambda: _return(_cuda(10, 8, dtype=torch.float64)),
    "rows on another GPU": lambda: _return(_cuda(10, 8, device="cuda:1")),
    "an order of 64 bits": lambda: _return(order=_order(dtype=torch.int64)),
    "an order of fewer experts": lambda: _return(order=_order()._replace(experts=5)),
    "an order in pieces": lambda: _return(order=_order()._replace(inverse=_cuda(2, 5, dtype=torch.int32).t())),
    "an order of two GPUs": lambda: _return(order=_order()._replace(offsets=_cuda(5, dtype=torch.int32,
                                                                                  device="cuda:1"))),
    "weights of another shape": lambda: _return(weights=_cuda(2, 5)),
    "weights of integers": lambda: _return(weights=_cuda(5, 2, dtype=torch.int32)),
    "residual of another type": lambda: _return(residual=_cuda(5, 8, dtype=F32)),
    "residual of other tokens": lambda: _return(residual=_cuda(4, 8)),
    "out of one row repeated": lambda: _return(out=_cuda(1, 8).expand(5, 8)),
    "out where gradients are recorded": lambda: _return(_cuda(10, 8).requires_grad_(), out=_cuda(5, 8)),
}


@pytest.mark.parametrize("what", list(LINEAR))
def test_linear_refuses(what):
    with FakeTensorMode(), pytest.raises(ValueError):
        LINEAR[what]()


@pytest.mark.parametrize("what", list(EXPERTS))
def test_experts_refuse(what):
    with FakeTensorMode(), pytest.raises(ValueError):
        EXPERTS[what]()


def test_empty_batches_reach_no_kernel():
    """No rows: the result's shape, and zero offsets, without a call."""
    with FakeTensorMode():
        assert _linear(_matrix(), _cuda(0, 64), activation="gelu_mul").shape == (0, 32)
        assert _linear(_matrix(), _cuda(2, 0, 64)).shape == (2, 0, 64)
        assert _grouped(_matrix(groups=2), _cuda(0, 64), _cuda(3, dtype=torch.int32)).shape == (0, 64)
        rows, order = _sort(_cuda(0, 8), _cuda(0, 2, dtype=torch.int32))
        assert rows.shape == (0, 8) and order.inverse.shape == (0, 2) and order.offsets.shape == (5,)
        assert _return(rows, order).shape == (0, 8)


@pytest.fixture(scope="module")
def lib():
    return load_library()


# A handle that only has to be there: every call below is refused on its numbers.
HANDLE = C.create_string_buffer(1 << 16)
P = C.addressof(HANDLE)


def _c_sort(lib, type=0, x_stride=8, tokens=5, hidden=8, ids_bytes=4, ids_stride=2, topk=2, n=4, rt=P, x=P, ids=P,
            offsets=P):
    return lib.nvfp4_expert_sort(rt, x, type, x_stride, tokens, hidden, ids, ids_bytes, ids_stride, topk, n, P, P, P,
                                 offsets, None)


def _c_return(lib, rows=P, type=0, rows_stride=8, weights=None, weights_type=0, residual=None, residual_stride=8,
              tokens=5, topk=2, hidden=8, out=P + 4096, out_stride=8, rt=P, inverse=P):
    return lib.nvfp4_expert_return(rt, rows, type, rows_stride, inverse, weights, weights_type, residual,
                                   residual_stride, tokens, topk, hidden, out, out_stride, None)


C_CALLS = {
    "sort without a runtime": lambda lib: _c_sort(lib, rt=None),
    "sort without x": lambda lib: _c_sort(lib, x=None),
    "sort without offsets": lambda lib: _c_sort(lib, offsets=None),
    "sort of an unknown type": lambda lib: _c_sort(lib, type=3),
    "sort of no tokens": lambda lib: _c_sort(lib, tokens=0),
    "sort of 2^31 picks": lambda lib: _c_sort(lib, tokens=1 << 30),
    "sort by 16-bit ids": lambda lib: _c_sort(lib, ids_bytes=2),
    "sort by 65 picks": lambda lib: _c_sort(lib, topk=65),
    "sort by 1025 experts": lambda lib: _c_sort(lib, n=1025),
    "sort with a negative stride": lambda lib: _c_sort(lib, x_stride=-8),
    "return without a runtime": lambda lib: _c_return(lib, rt=None),
    "return without an order": lambda lib: _c_return(lib, inverse=None),
    "return by weights of an unknown type": lambda lib: _c_return(lib, weights=P, weights_type=7),
    "return into rows that overlap": lambda lib: _c_return(lib, out_stride=7),
    "return onto its rows": lambda lib: _c_return(lib, out=P),
    "return onto its rows' end": lambda lib: _c_return(lib, out=P + 9 * 16 + 14),
    "return beside the residual": lambda lib: _c_return(lib, residual=P + 4096 + 16),
    "return on the residual in other steps": lambda lib: _c_return(lib, residual=P + 4096, residual_stride=16),
    "linear without a matrix": lambda lib: lib.nvfp4_linear_fused(P, None, P, 0, 64, 1, None, 0, 0, None, 0, P, 64, None,
                                                                  0, None),
    "grouped linear without a runtime": lambda lib: lib.nvfp4_linear_grouped(None, None, P, 0, 64, 1, P, None, 0, 0, P,
                                                                             64, 0, None, 0, None),
    "return's gradient of nothing": lambda lib: lib.nvfp4_expert_return_backward(
        P, P, 0, 8, None, 0, P, P, None, 0, 5, 2, 8, 4, None, None, None),
    "return's gradient without experts": lambda lib: lib.nvfp4_expert_return_backward(
        P, P, 0, 8, None, 0, P, P, None, 0, 5, 2, 8, 0, P, None, None),
    "upload without a runtime": lambda lib: lib.nvfp4_matrix_upload_grouped(None, P, 64, P, 8, P, 1, 2, 64,
                                                                            C.byref(C.c_void_p())),
    "upload of no groups": lambda lib: lib.nvfp4_matrix_upload_grouped(P, P, 64, P, 8, P, 0, 2, 64,
                                                                       C.byref(C.c_void_p())),
    "upload of 1025 groups": lambda lib: lib.nvfp4_matrix_upload_grouped(P, P, 64, P, 8, P, 1025, 2, 64,
                                                                         C.byref(C.c_void_p())),
    "upload of 2^31 rows": lambda lib: lib.nvfp4_matrix_upload_grouped(P, P, 64, P, 8, P, 1024, 1 << 21, 64,
                                                                       C.byref(C.c_void_p())),
    "upload of too few bytes": lambda lib: lib.nvfp4_matrix_upload_grouped(P, P, 63, P, 8, P, 1, 2, 64,
                                                                           C.byref(C.c_void_p())),
}


@pytest.mark.parametrize("what", list(C_CALLS))
def test_c_entry_refuses(lib, what):
    assert C_CALLS[what](lib) == 1
    assert lib.nvfp4_last_error()
