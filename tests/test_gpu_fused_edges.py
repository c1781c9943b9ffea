"""The NVFP4 linear with its epilogue and the expert sort and return at the edges of what they promise: ranges of values,
long rows, orders changed after the sort, calls one after the other (needs an sm_100a GPU)."""

from __future__ import annotations

import math

import numpy as np
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


# ------------------------------------------------------------------ an order changed after the sort


def _dropped(order, seed, share):
    """The order with some picks dropped after the sort, by a capacity limit say."""
    gen = torch.Generator().manual_seed(seed)
    gone = (torch.rand(order.inverse.shape, generator=gen) < share).cuda()
    return order._replace(inverse=torch.where(gone, -1, order.inverse))


def _return_gradients(order, g, rows, weights):
    """(drows, dweights) of the return by their formulas in 64 bits."""
    inverse, has = order.inverse.long(), order.inverse >= 0
    count = inverse.numel()
    drows = torch.zeros(count + 1, g.shape[1], dtype=torch.float64, device="cuda")
    drows[torch.where(has, inverse, count)] = weights.double()[..., None] * g.double()[:, None]
    taken = rows.double()[inverse.clamp(min=0)] * has[..., None]
    products = g.double()[:, None] * taken
    return drows[:-1], products.sum(2), products.abs().sum(2)


# The last one has more rows than one CTA marks at a time, the third fewer picks than threads.
@pytest.mark.parametrize("share", [0.3, 1.0])
@pytest.mark.parametrize("tokens,topk,experts,hidden", [(1, 1, 1, 8), (1, 8, 256, 40), (5, 3, 4, 33), (128, 8, 64, 96),
                                                        (700, 6, 1024, 20), (3001, 8, 256, 24), (40000, 8, 16, 2)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_gradients_of_picks_dropped_after_the_sort(cuda_runtime, kind, tokens, topk, experts, hidden, share):
    """A pick set to -1 after the sort is left out of the sum, and its row has a gradient of zero: whatever the memory
    of the gradient held, through autograd and at the C ABI, with every kind of output asked for."""
    from vllm_nvfp4_cuda.experts import TYPES as CODES, stream_of

    rt, dtype = cuda_runtime, TYPES[kind]
    gen = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, experts, (tokens, topk), generator=gen, dtype=torch.int32).cuda()
    rows, order = rt.expert_sort(_normal(81, tokens, hidden, dtype=dtype), ids, experts)
    order = _dropped(order, 82, share)
    weights, g = _normal(83, tokens, topk).requires_grad_(), _normal(84, tokens, hidden, dtype=dtype)
    want, dw, dw_size = _return_gradients(order, g, rows, weights.detach())
    half, unit, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -24, torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    tol, dw_tol = (unit * (1 + half) + half) * want.abs() + tiny, hidden * unit * dw_size + 2 * unit * dw.abs()
    rows = rows.requires_grad_()
    out = rt.expert_return(rows, order, weights)
    torch.full_like(rows, float("nan"))  # in the memory that the gradient gets next
    drows, dweights = torch.autograd.grad(out, (rows, weights), g)
    ref.check(drows, want, tol, "drows")
    ref.check(dweights, dw, dw_tol, "dweights")
    for with_weights in (True, False):
        for with_dweights in (True, False):
            drows, dweights = torch.full_like(g.new_empty(tokens * topk, hidden), float("nan")), torch.zeros_like(weights)
            status = rt.lib.nvfp4_expert_return_backward(
                rt.handle, g.data_ptr(), CODES[dtype], hidden, rows.data_ptr() if with_dweights else None, hidden,
                order.inverse.data_ptr(), order.offsets.data_ptr(), weights.data_ptr() if with_weights else None, 2,
                tokens, topk, hidden, experts, drows.data_ptr(), dweights.data_ptr() if with_dweights else None,
                stream_of(g.device))
            assert status == 0
            if with_weights:
                ref.check(drows, want, tol, "drows at the C ABI")
            else:
                named = want.abs().sum(1) > 0
                assert not bool(drows[~named].any()) and bool(drows[named].isfinite().all())
            if with_dweights:
                ref.check(dweights, dw, dw_tol, "dweights at the C ABI")


def test_captured_gradients_of_another_order(cuda_runtime):
    """Both passes captured once and replayed on orders with other picks dropped, none and all among them."""
    rt, tokens, topk, experts, hidden = cuda_runtime, 900, 6, 40, 72
    gen = torch.Generator().manual_seed(5)
    ids = torch.randint(0, experts, (tokens, topk), generator=gen, dtype=torch.int32).cuda()
    rows, sorted_order = rt.expert_sort(_normal(85, tokens, hidden), ids, experts)
    rows, weights = rows.requires_grad_(), _normal(86, tokens, topk).requires_grad_()
    g = _normal(87, tokens, hidden)
    order = sorted_order._replace(inverse=sorted_order.inverse.clone())

    def step():
        return torch.autograd.grad(rt.expert_return(rows, order, weights), (rows, weights), g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        drows, dweights = step()
    for share in (0.2, 0.0, 1.0, 0.01):
        order.inverse.copy_(_dropped(sorted_order, 88, share).inverse)
        want, dw, size = _return_gradients(order, g, rows.detach(), weights.detach())
        drows.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        ref.check(drows, want, 2.0 ** -24 * want.abs(), share)
        ref.check(dweights, dw, hidden * 2.0 ** -24 * size + 2.0 ** -23 * dw.abs(), share)


# ------------------------------------------------------------------ ranges of values


@pytest.mark.parametrize("vectors", [1, 4, 50])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_tiny_rows_and_large_divisors(cuda_runtime, kind, vectors):
    """Rows near the smallest normal numbers under divisors of real checkpoints: the results are normal numbers, and as
    many of their bits are right as elsewhere."""
    rt, dtype = cuda_runtime, TYPES[kind]
    packed, scales, _ = ref.random_matrix(2, 70, 256, 90)
    divisors = torch.tensor([9e3, 1.1e5])
    m = rt.upload_grouped(packed.cuda(), scales.cuda(), divisors.cuda())
    one = rt.upload_grouped(packed[1:].cuda(), scales[1:].cuda(), divisors[1:].cuda())
    for size in (1e-32, 1e-34):
        x = (_normal(91, vectors, 256).double() * size).to(dtype)
        bias = (_normal(92, 70).double() * size * 1e-4).float()
        want, tol = ref.linear(x, packed[1].cuda(), scales[1].cuda(), divisors[1].cuda(), bias)
        assert float(want.abs().median()) > 2.0 ** -126
        ref.check(rt.linear_fused(one, x, bias=bias), want, tol, size)
        offsets = torch.tensor([0, 0, vectors], dtype=torch.int32, device="cuda")
        both = torch.stack([bias, bias])
        ref.check(rt.linear_grouped(m, x, offsets, bias=both), want, tol, size)
    m.close()
    one.close()


@pytest.mark.parametrize("vectors", [1, 6, 50])
def test_bits_of_fp32_elements(cuda_runtime, vectors):
    """Elements of an FP32 row are right to 2^-23 of themselves, or to 2^-39 of the row's largest value where that is
    more (from 2^-16 of it down): shown with the largest value in columns whose weights are zero."""
    rt, rows, cols = cuda_runtime, 48, 160
    packed, scales, divisors = ref.random_matrix(1, rows, cols, 93)
    packed[:, :, :8] = 0  # the first 16 columns
    m = rt.upload_grouped(packed.cuda(), scales.cuda(), divisors.cuda())
    w = ref.weights(packed[0], scales[0]).cuda()
    inv = (1.0 / divisors.cuda()).double()
    for largest in (1.0, 2.0 ** 15, 2.0 ** 20, 2.0 ** 29):
        x = _normal(94, vectors, cols)
        x[:, 3] = largest
        got = rt.linear_fused(m, x).double()
        xd = x.double()
        element = torch.maximum(xd.abs() * 2.0 ** -23, xd.abs().amax(1, keepdim=True) * 2.0 ** -39)
        _, tol = ref.linear(x[:, 16:], packed[0, :, 8:].cuda(), scales[0, :, 1:].cuda(), divisors[0].cuda())
        ref.check(got, xd @ w.t() * inv, tol + element @ w.abs().t() * inv, largest)
    m.close()


@pytest.mark.parametrize("cols", [4112, 8192, 11008, 49152])
@pytest.mark.parametrize("vectors", [3, 40, 200])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_long_sums_of_one_sign(cuda_runtime, kind, vectors, cols):
    """Products of one sign over long rows, the rounded sum taken off again by the residual, so that what is left shows
    the FP32 sum itself: low by less than 2^-14 of it (an eighth of FP16's half step) whatever the length, and the bits
    of a second call."""
    rt, dtype, rows = cuda_runtime, TYPES[kind], 301
    packed, scales, divisors = ref.random_matrix(2, rows, cols, 95)
    packed &= 0x77  # no weight below zero
    divisors = divisors * (cols / 64)
    m = rt.upload_grouped(packed[:1].cuda(), scales[:1].cuda(), divisors[:1].cuda())
    gen = torch.Generator().manual_seed(96)
    x = torch.rand(vectors, cols, generator=gen).to(dtype).cuda()
    z = x.double() @ ref.weights(packed[0].cuda(), scales[0].cuda()).t() * (1.0 / divisors[0]).double().cuda()
    taken = (-z).to(dtype)
    want = z + taken.double()
    half = torch.finfo(dtype).eps / 2
    got = rt.linear_fused(m, x, residual=taken)
    ref.check(got, want, 2.0 ** -14 * z * (1 + half) + half * want.abs() + torch.finfo(dtype).tiny)
    assert torch.equal(got, rt.linear_fused(m, x, residual=taken))
    m.close()
    # The same sums with a gate over groups of uneven rows, against the plain bound of the type.
    m = rt.upload_grouped(packed[:, :300].contiguous().cuda(), scales[:, :300].contiguous().cuda(), divisors.cuda())
    cut = vectors // 3
    offsets = torch.tensor([0, cut, vectors], dtype=torch.int32, device="cuda")
    got = rt.linear_grouped(m, x, offsets, activation="relu_mul")
    for g, rows_of in enumerate((slice(0, cut), slice(cut, vectors))):
        w = ref.weights(packed[g, :300].cuda(), scales[g, :300].cuda())
        z = x[rows_of].double() @ w.t() * (1.0 / divisors[g]).double().cuda()
        want = z[:, :150] * z[:, 150:]
        ref.check(got[rows_of], want, (2.0 ** -13 + 2.0 ** -20 + half) * want)
    m.close()


@pytest.mark.parametrize("vectors", [8, 640])
def test_fp32_activations_to_their_last_bits(cuda_runtime, vectors):
    """SiLU and GELU's tanh form of FP32 rows against 64 bits, relative to the result: exp and the fast division (by 1 to
    2) are off by two units at most (2^-23 each), the sum and a product by half of one each: five. The tanh form's
    argument u, whose error exp passes on, takes half a unit for its factor, its last product and the FMA each, and for
    three more roundings of the cubic part: six halves of a unit of u."""
    rt = cuda_runtime
    # The identity: code 2 is 1, scale byte 0x38 is 1.
    packed = torch.zeros(1, 16, 8, dtype=torch.uint8)
    for r in range(16):
        packed[0, r, r // 2] = 2 << (4 * (r % 2))
    m = rt.upload_grouped(packed.cuda(), torch.full((1, 16, 1), 0x38, dtype=torch.uint8).cuda(), torch.ones(1).cuda())
    for name, low in (("silu", -87.0), ("gelu_tanh", -9.0)):
        x = torch.linspace(low, 20.0, vectors * 16).reshape(vectors, 16).cuda()
        z = rt.linear_fused(m, x).double()  # what the activation gets
        u = z if name == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        want = z * torch.sigmoid(u)
        units = 5.0 if name == "silu" else 5.0 + 3.0 * u.abs()
        ref.check(rt.linear_fused(m, x, activation=name), want, units * 2.0 ** -23 * want.abs() + 2.0 ** -149, name)
        up = rt.upload_grouped(packed.repeat(1, 2, 1).cuda(), torch.full((1, 32, 1), 0x38, dtype=torch.uint8).cuda(),
                               torch.ones(1).cuda())
        ref.check(rt.linear_fused(up, x, activation=name + "_mul"), want * z, (units + 0.5) * 2.0 ** -23 * (want * z).abs()
                  + 2.0 ** -140, name)
        up.close()
    m.close()


# ------------------------------------------------------------------ what a call does to its tensors


def test_forward_mode_derivatives_of_gradients_are_refused(cuda_runtime):
    """A tangent that comes in with the gradient of the sort or the return would be dropped."""
    from torch.autograd import forward_ad

    ids = torch.tensor([[0], [1], [0]], dtype=torch.int32, device="cuda")
    x = _normal(101, 3, 8).requires_grad_()
    rows, order = cuda_runtime.expert_sort(x, ids, 2)
    out = cuda_runtime.expert_return(rows, order)
    with forward_ad.dual_level():
        for result in (rows, out):
            g = forward_ad.make_dual(torch.ones_like(result), torch.ones_like(result))
            with pytest.raises(ValueError, match="forward-mode"):
                torch.autograd.grad(result, x, g, retain_graph=True)
    (dx,) = torch.autograd.grad(out, x, torch.ones_like(out))
    assert torch.equal(dx, torch.ones_like(x))


def test_writing_to_out_is_seen_by_autograd(cuda_runtime):
    """A tensor that autograd keeps for a gradient and that a call then writes to as its out: the backward pass says so,
    as after any other operation in place."""
    rt = cuda_runtime
    packed, scales, divisors = ref.random_matrix(2, 32, 32, 97)
    one = rt.upload_grouped(packed[:1].cuda(), scales[:1].cuda(), divisors[:1].cuda())
    two = rt.upload_grouped(packed.cuda(), scales.cuda(), divisors.cuda())
    x = _normal(98, 6, 32)
    ids = torch.tensor([[0], [1], [0], [0], [1], [1]], dtype=torch.int32, device="cuda")
    rows, order = rt.expert_sort(x, ids, 2)
    calls = [lambda out: rt.linear_fused(one, x, out=out),
             lambda out: rt.linear_fused(one, x.view(2, 3, 32), out=out.view(2, 3, 32)),
             lambda out: rt.linear_grouped(two, rows, order.offsets, out=out),
             lambda out: rt.expert_return(rows, order, out=out),
             lambda out: rt.linear_fused(one, x[:0], out=out[:0])]
    for i, call in enumerate(calls):
        scale, kept = torch.ones(1, device="cuda", requires_grad=True), _normal(99, 6, 32)
        value = (scale * kept).sum()
        call(kept)
        if i < 4:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                value.backward()
        else:  # nothing was written
            value.backward()
    with torch.inference_mode():
        out = torch.empty(6, 32, device="cuda")
        assert rt.linear_fused(one, x, out=out) is out
    one.close()
    two.close()


def test_divisors_of_zero_are_refused(cuda_runtime):
    """As the dense upload refuses one: from host and device memory, wherever in the list it stands."""
    packed, scales, divisors = ref.random_matrix(3, 16, 32, 100)
    for at in range(3):
        bad = divisors.clone()
        bad[at] = 0.0
        with pytest.raises(RuntimeError, match="divisor"):
            cuda_runtime.upload_grouped(packed.numpy(), scales.numpy(), bad.numpy())
        with pytest.raises(RuntimeError, match="divisor"):
            cuda_runtime.upload_grouped(packed.cuda(), scales.cuda(), bad.cuda())
    cuda_runtime.upload_grouped(packed.numpy(), scales.numpy(), divisors.numpy()).close()


# ------------------------------------------------------------------ many picks, far addresses


def _plain_order(ids, experts):
    """perm, inverse and offsets of a stable sort, on the host."""
    flat = ids.reshape(-1).astype(np.int64)
    kept = np.flatnonzero((flat >= 0) & (flat < experts))
    picks = kept[np.argsort(flat[kept], kind="stable")]
    perm, inverse = np.full(flat.size, -1), np.full(flat.size, -1)
    perm[:picks.size] = picks
    inverse[picks] = np.arange(picks.size)
    return perm, inverse.reshape(ids.shape), np.concatenate(([0], np.cumsum(np.bincount(flat[kept], minlength=experts))))


@pytest.mark.parametrize("how", ["all", "some", "one", "runs"])
@pytest.mark.parametrize("tokens,topk,experts,hidden", [(8192, 8, 256, 4), (9001, 8, 256, 4), (70001, 1, 9, 1),
                                                        (66000, 2, 1024, 3), (33000, 8, 16, 8)])
def test_order_of_many_picks(cuda_runtime, tokens, topk, experts, hidden, how):
    """More picks than the ranking cluster's warps hold at a time (65,536): the stable order, each time."""
    rng = np.random.default_rng(tokens + topk)
    ids = rng.integers(0, experts, size=(tokens, topk))
    if how == "one":
        ids[:] = experts - 1
    elif how == "some":
        ids[rng.random(ids.shape) < 0.3] = experts + 5
    elif how == "runs":  # picks of a warp all alike, those of the next another expert's
        ids = (np.arange(tokens * topk) // 640 % experts).reshape(tokens, topk)
    perm, inverse, offsets = _plain_order(ids, experts)
    x = _normal(110, tokens, hidden, dtype=torch.bfloat16)
    for _ in range(2):
        rows, order = cuda_runtime.expert_sort(x, torch.from_numpy(ids.astype(np.int32)).cuda(), experts)
        np.testing.assert_array_equal(order.perm.cpu().numpy(), perm)
        np.testing.assert_array_equal(order.inverse.cpu().numpy(), inverse)
        np.testing.assert_array_equal(order.offsets.cpu().numpy(), offsets)
        used = int(offsets[-1])
        assert torch.equal(rows[:used], x[torch.from_numpy(perm[:used] // topk).cuda()]) and not bool(rows[used:].any())


def test_row_strides_past_32_bits(cuda_runtime):
    """Rows so far apart that their places pass 2^32 bytes and 2^31 elements, read and written by every operator."""
    rt, step = cuda_runtime, 260_000_008
    far = torch.zeros(11 * step + 256, dtype=torch.bfloat16, device="cuda")
    assert far.numel() > 2 ** 31
    packed, scales, divisors = ref.random_matrix(1, 40, 48, 111)
    m = rt.upload_grouped(packed.cuda(), scales.cuda(), divisors.cuda())
    ids = torch.tensor([[i % 3] for i in range(12)], dtype=torch.int32, device="cuda")
    for rows in (7, 12):
        x, out = far.as_strided((rows, 48), (step, 1)), far.as_strided((rows, 40), (step, 1), 48 + 8)
        x.copy_(_normal(112, rows, 48, dtype=torch.bfloat16))
        want, tol = ref.linear(x.contiguous(), packed[0].cuda(), scales[0].cuda(), divisors[0].cuda())
        for start in (0, 1):  # where TMA can read the rows, and where it cannot
            y = x if start == 0 else far.as_strided((rows, 48), (step, 1), 1).copy_(x.clone())
            ref.check(rt.linear_fused(m, y, out=out), want, tol)
            out.zero_()
            offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
            ref.check(rt.linear_grouped(m, y, offsets, out=out), want, tol)
            near, order = rt.expert_sort(y, ids[:rows], 3)
            assert torch.equal(near, y[order.perm.long()])
            back = rt.expert_return(y, order, out=far.as_strided((rows, 48), (step, 1), 104))
            assert torch.equal(back, y[order.inverse[:, 0].long()])
    m.close()


def test_results_past_32_bits(cuda_runtime):
    """More than 2^31 outputs of one call, the first and the last of them looked at."""
    rt, rows, vectors = cuda_runtime, 140_000, 15_500
    packed, scales, divisors = ref.random_matrix(1, rows, 16, 113)
    m = rt.upload_grouped(packed.cuda(), scales.cuda(), divisors.cuda())
    x = _normal(114, vectors, 16, dtype=torch.float16)
    out = rt.linear_fused(m, x)
    assert out.numel() > 2 ** 31
    for v in (slice(0, 70), slice(-70, None)):
        for r in (slice(0, 300), slice(rows - 300, rows)):
            want, tol = ref.linear(x[v], packed[0, r].cuda(), scales[0, r].cuda(), divisors[0].cuda())
            ref.check(out[v, r], want, tol)
    m.close()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_long_rows_over_several_tiles_a_pair(cuda_runtime, kind):
    """Rows of several segments where every pair of CTAs has several tiles, dense with a residual and over groups of uneven
    rows: the bits of calls of one tile a pair, which are right to the plain bound."""
    rt, dtype, cols = cuda_runtime, TYPES[kind], 8208
    half = torch.finfo(dtype).eps / 2
    gen = torch.Generator(device="cuda").manual_seed(115)

    def matrix(groups, rows):
        packed = torch.randint(0, 256, (groups, rows, cols // 2), generator=gen, dtype=torch.uint8, device="cuda")
        scales = torch.randint(0x28, 0x48, (groups, rows, cols // 16), generator=gen, dtype=torch.uint8, device="cuda")
        divisors = torch.rand(groups, generator=gen, device="cuda") * 2000 + 3000
        return rt.upload_grouped(packed, scales, divisors), packed, scales, divisors

    def near(got, x, packed, scales, divisor, residual=None):
        w = ref.weights(packed, scales)
        z, size = x.double() @ w.t() / divisor.double(), x.double().abs() @ w.abs().t() / divisor.double()
        z = z if residual is None else z + residual.double()
        # A chain's truncations are of its running sum, which is far below the sum of sizes; the divisor's inverse is FP32.
        ref.check(got, z, half * z.abs() * (1 + half) + 2.0 ** -14 * size + torch.finfo(dtype).tiny)

    rows, vectors = 5000, 900  # 20 pairs of weight tiles, six tiles of rows: 120 items for 74 pairs
    m, packed, scales, divisors = matrix(1, rows)
    x, residual = _normal(116, vectors, cols, dtype=dtype), _normal(117, vectors, rows, dtype=dtype)
    out = rt.linear_fused(m, x, residual=residual)
    for v in range(0, vectors, 150):
        part = slice(v, v + 150)
        assert torch.equal(out[part], rt.linear_fused(m, x[part], residual=residual[part]))
    near(out[:150, :700], x[:150], packed[0, :700], scales[0, :700], divisors[0], residual[:150, :700])
    m.close()
    groups, counts = 8, [0, 1, 300, 0, 161, 17, 160, 500]
    m, packed, scales, divisors = matrix(groups, 1400)
    offsets = [0, *np.cumsum(counts).tolist()]
    x = _normal(118, offsets[-1] + 4, cols, dtype=dtype)
    out = rt.linear_grouped(m, x, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    assert not bool(out[offsets[-1]:].any())
    for g, count in enumerate(counts):
        part = slice(offsets[g], offsets[g + 1])
        one = rt.upload_grouped(packed[g:g + 1], scales[g:g + 1], divisors[g:g + 1])
        if count > 8:
            assert torch.equal(out[part], rt.linear_fused(one, x[part]))
        if count:
            near(out[part], x[part], packed[g], scales[g], divisors[g])
        one.close()
    m.close()
