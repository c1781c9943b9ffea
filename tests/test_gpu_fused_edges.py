"""The NVFP4 linear with its epilogue and the expert sort and return at the edges of what they promise: ranges of values,
long rows, orders changed after the sort, calls one after the other (needs an sm_100a GPU)."""

from __future__ import annotations

import pytest
import torch

import fused_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _normal(seed, *shape, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


@pytest.mark.parametrize("kind", list(TYPES))
def test_short_calls_one_after_the_other(cuda_runtime, kind):
    """Calls of the many-row kernel that are over after one step of columns, each followed at once by kernels that take
    over the shared memory of its CTAs: the bits of the first call, every time."""
    rt, dtype = cuda_runtime, TYPES[kind]
    packed, scales, divisors = ref.random_matrix(1, 700, 64, 70)
    m = rt.upload_grouped(packed.cuda(), scales.cuda(), divisors.cuda())
    many, few = _normal(71, 40, 64, dtype=dtype), _normal(72, 2, 64, dtype=dtype)
    want_many, want_few = rt.linear_fused(m, many), rt.linear_fused(m, few)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(60):
        got.append((rt.linear_fused(m, many), rt.linear_fused(m, few), rt.linear_fused(m, many, stream=side)))
    torch.cuda.synchronize()
    for a, b, c in got:
        assert torch.equal(a, want_many) and torch.equal(b, want_few) and torch.equal(c, want_many)
    rt.synchronize()
    m.close()
