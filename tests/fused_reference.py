"""The NVFP4 linear with its epilogue in 64 bits, and how far a kernel may be from it (host-side, torch float64).

Tolerance of one product: the kernels add exact products in FP32 chains on tensor cores, which round the running sum
(towards zero at worst: one unit of 2^-23 of the larger of the sum and the products) once per 16 columns, per
activation term. With P the largest running sum at a multiple of 16 columns plus the largest sum of absolute products
of 16 columns, a chain of n steps is off by at most n * 2^-23 * P. FP32 activations enter as two halves (off by at
most 2^-23 of an element) or three parts. The chain may be cut anywhere, which only shortens it. The epilogue's
operations add a few units of 2^-24 of their results, and the output's rounding half a step of its type.
"""

from __future__ import annotations

import math

import torch

E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
UNIT = 2.0 ** -24


def random_matrix(groups, rows, cols, seed):
    """Codes and scale bytes of every kind: (packed, scales, divisors) on the CPU; scales include zero, subnormal and
    the largest values, divisors differ by group."""
    gen = torch.Generator().manual_seed(seed)
    packed = torch.randint(0, 256, (groups, rows, cols // 2), generator=gen, dtype=torch.uint8)
    scales = torch.randint(0x28, 0x48, (groups, rows, cols // 16), generator=gen, dtype=torch.uint8)
    odd = torch.randint(0, 0x7F, scales.shape, generator=gen, dtype=torch.uint8)
    scales = torch.where(torch.rand(scales.shape, generator=gen) < 0.02, odd, scales)
    divisors = torch.rand(groups, generator=gen) * 30 + 20
    return packed, scales, divisors


def weights(packed, scales):
    """float64 [..., rows, cols], without the divisor."""
    b = scales.to(torch.int64)
    e, m = b >> 3, (b & 7).double()
    s = torch.where(e == 0, m / 512, (1 + m / 8) * torch.exp2((e - 7).double()))
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).long()
    return E2M1.to(packed.device)[codes] * s.repeat_interleave(16, dim=-1)


def _product(x, w):
    """x w^T and P of the module docstring, float64 [vectors, rows]."""
    v, k = x.shape
    n = k // 16
    xb, wb = x.reshape(v, n, 16), w.reshape(-1, n, 16)
    blocks = torch.einsum("vnk,rnk->vrn", xb, wb)
    size = torch.einsum("vnk,rnk->vrn", xb.abs(), wb.abs())
    runs = blocks.cumsum(-1)
    return runs[..., -1], runs.abs().amax(-1) + size.amax(-1), size.sum(-1)


def linear(x, packed, scales, divisor, bias=None, activation=None, residual=None):
    """(reference, tolerance) float64 [vectors, width] of one group; x etc. as the kernel gets them."""
    inv = (1.0 / divisor.float()).double()  # the kernel multiplies by the FP32 inverse
    z, p, size = _product(x.double(), weights(packed, scales))
    steps = x.shape[1] // 16 * (3 if x.dtype == torch.float32 else 1) + 16
    err = (steps * 2 * UNIT * p + 2 * UNIT * size) * inv
    z = z * inv
    err = err + 4 * UNIT * z.abs()
    if bias is not None:
        z = z + bias.double()
        err = err + UNIT * z.abs()
    if activation:
        gated = activation.endswith("_mul")
        base = activation[:-4] if gated else activation
        up = None
        if gated:
            half = z.shape[1] // 2
            z, up, err, err_up = z[:, :half], z[:, half:], err[:, :half], err[:, half:]
        if base == "relu":
            y = z.clamp(min=0)
        elif base == "silu":
            y = z * torch.sigmoid(z)
        elif base == "gelu":
            y = z * torch.special.ndtr(z)
        else:
            y = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        # The slopes stay below 1.13; exp, erfc, the division and the cubic's argument (whose rounding grows with the
        # argument, where the result is small) are off by a few units of the result and of z.
        err = 1.13 * err + 16 * UNIT * (y.abs() + z.abs())
        if gated:
            err = err * up.abs() + err_up * y.abs() + err * err_up + UNIT * (y * up).abs()
            y = y * up
        z = y
    if residual is not None:
        z = z + residual.double()
        err = err + UNIT * z.abs()
    # Half a step of the type, and of its smallest normal number below that (FP16).
    info = torch.finfo(x.dtype)
    tol = err + info.eps / 2 * (z.abs() + err) + info.tiny * info.eps
    # Rounding to the type takes a value that is half a step past its largest number, or more, to infinity (FP16:
    # from 65520 on).
    over = z.abs() - err >= info.max * (1 + info.eps / 4)
    return torch.where(over, torch.copysign(torch.full_like(z, math.inf), z), z), tol


def check(got, want, tolerance, what=""):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = torch.where(got == want, 0.0, (got - want).abs())  # infinities equal themselves
    bad = ~(off <= tolerance)
    assert not bool(bad.any()), (what, int(bad.sum()), float((off / tolerance).max()), bad.nonzero()[:4].tolist())
