"""Calls of the fused linears and the expert sort and return that the checks before any kernel have to refuse, beside those
of test_fused_refusals.py (no GPU)."""

from __future__ import annotations

import ctypes as C
from types import SimpleNamespace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

from vllm_nvfp4_cuda import experts, fused
from vllm_nvfp4_cuda.runtime import load_library


@pytest.fixture(scope="module")
def lib():
    return load_library()


# A handle that only has to be there: every call below is refused on its numbers. The rest stands for device memory,
# of which only the addresses are looked at.
HANDLE = C.create_string_buffer(1 << 16)
P = (C.addressof(HANDLE) + 255) & ~255
BF16, F16, F32 = 0, 1, 2


def _sort(lib, type=BF16, x=P, ids=P, ids_bytes=4, rows=P, perm=P, inverse=P, offsets=P):
    return lib.nvfp4_expert_sort(P, x, type, 8, 5, 8, ids, ids_bytes, 2, 2, 4, rows, perm, inverse, offsets, None)


def _return(lib, type=BF16, rows=P, inverse=P, weights=None, weights_type=F32, residual=None, out=P + 4096):
    return lib.nvfp4_expert_return(P, rows, type, 8, inverse, weights, weights_type, residual, 8, 5, 2, 8, out, 8, None)


def _gradient(lib, type=BF16, dout=P, rows=P, inverse=P, offsets=P, weights=P, weights_type=F32, drows=P + 4096,
              dweights=P + 8192):
    return lib.nvfp4_expert_return_backward(P, dout, type, 8, rows, 8, inverse, offsets, weights, weights_type, 5, 2, 8,
                                            4, drows, dweights, None)


# Addresses off their elements: a kernel that took one would fault.
MISALIGNED = {
    "sort of BF16 x": lambda lib: _sort(lib, x=P + 1),
    "sort of FP32 x": lambda lib: _sort(lib, type=F32, x=P + 2),
    "sort to rows": lambda lib: _sort(lib, type=F16, rows=P + 1),
    "sort by ids of 4 bytes": lambda lib: _sort(lib, ids=P + 2),
    "sort by ids of 8 bytes": lambda lib: _sort(lib, ids=P + 4, ids_bytes=8),
    "sort to perm": lambda lib: _sort(lib, perm=P + 1),
    "sort to inverse": lambda lib: _sort(lib, inverse=P + 2),
    "sort to offsets": lambda lib: _sort(lib, offsets=P + 2),
    "return of BF16 rows": lambda lib: _return(lib, rows=P + 1),
    "return of FP32 rows": lambda lib: _return(lib, type=F32, rows=P + 2),
    "return to out": lambda lib: _return(lib, type=F16, out=P + 4097),
    "return by inverse": lambda lib: _return(lib, inverse=P + 2),
    "return by FP32 weights": lambda lib: _return(lib, weights=P + 2),
    "return by BF16 weights": lambda lib: _return(lib, weights=P + 1, weights_type=BF16),
    "return onto a residual": lambda lib: _return(lib, residual=P + 8193),
    "gradient of dout": lambda lib: _gradient(lib, dout=P + 1),
    "gradient of rows": lambda lib: _gradient(lib, rows=P + 1),
    "gradient by inverse": lambda lib: _gradient(lib, inverse=P + 1),
    "gradient by offsets": lambda lib: _gradient(lib, offsets=P + 2),
    "gradient by weights": lambda lib: _gradient(lib, weights=P + 2),
    "gradient to drows": lambda lib: _gradient(lib, drows=P + 4097),
    "gradient to FP32 drows": lambda lib: _gradient(lib, type=F32, drows=P + 4098),
    "gradient to dweights": lambda lib: _gradient(lib, dweights=P + 8194),
}


@pytest.mark.parametrize("what", list(MISALIGNED))
def test_misaligned_addresses_are_refused(lib, what):
    assert MISALIGNED[what](lib) == 1
    assert b"aligned" in lib.nvfp4_last_error()


# ------------------------------------------------------------------ tensors without memory: the Python checks


class _Unreached:
    """Stands for the runtime: a call that is refused in time never asks it for anything."""

    def __getattr__(self, name):
        raise AssertionError(f"the runtime was reached ({name})")


RT = _Unreached()


def _cuda(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda:0")


def _matrix(rows=64, cols=64, groups=1):
    return SimpleNamespace(rows=rows, cols=cols, groups=groups, device=0)


def _order(tokens=5, topk=2, n=4):
    return experts.ExpertOrder(_cuda(tokens * topk, dtype=torch.int32), _cuda(tokens, topk, dtype=torch.int32),
                               _cuda(n + 1, dtype=torch.int32), n)


def _dual(*shape):
    return forward_ad.make_dual(_cuda(*shape), _cuda(*shape))


DUALS = {
    "linear of x": lambda: fused.linear_fused(RT, _matrix(), _dual(3, 64), None, None, None, None, None),
    "linear of bias": lambda: fused.linear_fused(RT, _matrix(), _cuda(3, 64), _dual(64), None, None, None, None),
    "linear of residual": lambda: fused.linear_fused(RT, _matrix(), _cuda(3, 64), None, None, _dual(3, 64), None, None),
    "grouped linear of x": lambda: fused.linear_grouped(RT, _matrix(groups=2), _dual(3, 64),
                                                        _cuda(3, dtype=torch.int32), None, None, None, None),
    "grouped linear of bias": lambda: fused.linear_grouped(RT, _matrix(groups=2), _cuda(3, 64),
                                                           _cuda(3, dtype=torch.int32), _dual(2, 64), None, None, None),
    "sort of x": lambda: experts.expert_sort(RT, _dual(5, 8), _cuda(5, 2, dtype=torch.int32), 4),
    "return of rows": lambda: experts.expert_return(RT, _dual(10, 8), _order()),
    "return of weights": lambda: experts.expert_return(RT, _cuda(10, 8), _order(), _dual(5, 2)),
    "return of residual": lambda: experts.expert_return(RT, _cuda(10, 8), _order(), None, _dual(5, 8)),
}


@pytest.mark.parametrize("what", list(DUALS))
def test_forward_mode_derivatives_are_refused(what):
    """A tangent would be dropped without a word; a dual level without tangents, or no_grad within one, changes nothing."""
    with FakeTensorMode(), forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            DUALS[what]()
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            DUALS[what]()


def test_calls_in_a_dual_level_without_tangents():
    with FakeTensorMode(), forward_ad.dual_level():
        assert fused.linear_fused(RT, _matrix(), _cuda(0, 64), None, None, None, None, None).shape == (0, 64)
        rows, order = experts.expert_sort(RT, _cuda(0, 8), _cuda(0, 2, dtype=torch.int32), 4)
        assert experts.expert_return(RT, rows, order).shape == (0, 8)


def _repeated(rows, columns, dtype=torch.bfloat16):
    return _cuda(1, columns, dtype=dtype).expand(rows, columns)


# Numbers that pass what the C ABI takes: an int of it would hold the low 32 bits, 3 or 8 here, and the call would do a
# part of the work.
HUGE = {
    "linear of 2^32 + 3 rows": lambda: fused.linear_fused(RT, _matrix(1, 16), _repeated(2 ** 32 + 3, 16), None, None, None,
                                                          None, None),
    "linear of 2^30 + 1 rows": lambda: fused.linear_fused(RT, _matrix(1, 16), _repeated(2 ** 30 + 1, 16), None, None, None,
                                                          None, None),
    "linear of 2^32 + 3 rows of three axes": lambda: fused.linear_fused(
        RT, _matrix(1, 16), _cuda(1, 1, 16).expand(2, 2 ** 31 + 2, 16), None, None, None, None, None),
    "grouped linear of 2^32 + 3 rows": lambda: fused.linear_grouped(
        RT, _matrix(1, 16, 2), _repeated(2 ** 32 + 3, 16), _cuda(3, dtype=torch.int32), None, None, None, None),
    "sort of 2^32 + 3 tokens": lambda: experts.expert_sort(RT, _repeated(2 ** 32 + 3, 1),
                                                           _repeated(2 ** 32 + 3, 1, torch.int32), 4),
    "sort of 2^31 picks": lambda: experts.expert_sort(RT, _repeated(2 ** 30, 1), _repeated(2 ** 30, 2, torch.int32), 4),
    "sort of 2^32 + 8 columns": lambda: experts.expert_sort(RT, _cuda(1, 2 ** 32 + 8), _cuda(1, 1, dtype=torch.int32), 4),
    "return of 2^32 + 3 tokens": lambda: experts.expert_return(RT, _repeated(2 ** 32 + 3, 1), _order(2 ** 32 + 3, 1)),
    "return of 2^32 + 8 columns": lambda: experts.expert_return(RT, _cuda(1, 2 ** 32 + 8), _order(1, 1)),
}


@pytest.mark.parametrize("what", list(HUGE))
def test_numbers_past_the_c_abi_are_refused(what):
    with FakeTensorMode(), pytest.raises(ValueError, match="at most"):
        HUGE[what]()


ELSEWHERE = SimpleNamespace(device=torch.device("cuda:1"), cuda_stream=0)  # of a stream, all that is looked at here
STREAMS = {
    "linear": lambda: fused.linear_fused(RT, _matrix(), _cuda(0, 64), None, None, None, None, ELSEWHERE),
    "grouped linear": lambda: fused.linear_grouped(RT, _matrix(), _cuda(0, 64), _cuda(2, dtype=torch.int32), None, None, None,
                                                   ELSEWHERE),
    "sort": lambda: experts.expert_sort(RT, _cuda(0, 8), _cuda(0, 2, dtype=torch.int32), 4, ELSEWHERE),
    "return": lambda: experts.expert_return(RT, _cuda(0, 8), _order(0), stream=ELSEWHERE),
}


@pytest.mark.parametrize("what", list(STREAMS))
def test_a_stream_of_another_gpu_is_refused(what):
    """The work would run on the current stream of the tensors' GPU instead, in no order with the given one."""
    with FakeTensorMode(), pytest.raises(ValueError, match="stream"):
        STREAMS[what]()
