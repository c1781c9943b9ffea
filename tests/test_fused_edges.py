"""Calls of the fused linears and the expert sort and return that the checks before any kernel have to refuse, beside those
of test_fused_refusals.py (no GPU)."""

from __future__ import annotations

import ctypes as C

import pytest

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
