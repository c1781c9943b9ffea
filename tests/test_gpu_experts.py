"""Rows sorted by expert and brought back (Runtime.expert_sort, Runtime.expert_return) and their gradients, against
their formulas in 64 bits, and the run of both around grouped products (needs an sm_100a GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import fused_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNIT = 2.0 ** -24


def _normal(seed, *shape, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def _ids(seed, tokens, topk, experts, how):
    rng = np.random.default_rng(seed)
    if how == "none":  # every pick dropped, by numbers on both sides
        return rng.choice([-1, experts, 2 ** 31 - 1, -2 ** 31], size=(tokens, topk)).astype(np.int32)
    ids = rng.integers(0, experts, size=(tokens, topk))  # the same expert twice in a token now and then
    if how == "one":
        ids[:] = experts - 1
    if how == "some":
        ids[rng.random(ids.shape) < 0.3] = -1
    return ids.astype(np.int32)


def _plain_order(ids, experts):
    flat = ids.reshape(-1).astype(np.int64)
    kept = np.flatnonzero((flat >= 0) & (flat < experts))
    picks = kept[np.argsort(flat[kept], kind="stable")]
    perm = np.full(flat.size, -1)
    perm[:picks.size] = picks
    inverse = np.full(flat.size, -1)
    inverse[picks] = np.arange(picks.size)
    offsets = np.concatenate(([0], np.cumsum(np.bincount(flat[kept], minlength=experts))))
    return perm, inverse.reshape(ids.shape), offsets


# tokens x topk on both sides of the one-CTA sort (4096 picks), with most experts and picks in each.
SIZES = [(1, 1, 1, 8), (1, 8, 256, 2048), (3, 2, 8, 1), (7, 64, 40, 33), (128, 8, 64, 96), (129, 8, 256, 100),
         (513, 6, 1024, 20), (700, 3, 5, 2052), (2048, 1, 3, 7), (3001, 8, 256, 24), (512, 8, 9, 4),
         (4097, 1, 1024, 8), (600, 64, 1024, 12)]


@pytest.mark.parametrize("how", ["all", "some", "none", "one"])
@pytest.mark.parametrize("tokens,topk,experts,hidden", SIZES)
def test_sort_and_its_gradient(cuda_runtime, tokens, topk, experts, hidden, how):
    ids = _ids(tokens + topk, tokens, topk, experts, how)
    perm, inverse, offsets = _plain_order(ids, experts)
    for kind, dtype in TYPES.items():
        x = _normal(1, tokens, hidden, dtype=dtype).requires_grad_()
        rows, order = cuda_runtime.expert_sort(x, torch.from_numpy(ids).cuda(), experts)
        np.testing.assert_array_equal(order.perm.cpu().numpy(), perm)
        np.testing.assert_array_equal(order.inverse.cpu().numpy(), inverse)
        np.testing.assert_array_equal(order.offsets.cpu().numpy(), offsets)
        used = int(offsets[-1])
        at = torch.from_numpy(perm[:used] // topk).cuda()
        assert torch.equal(rows[:used], x.detach()[at]) and not bool(rows[used:].any())
        g = _normal(2, tokens * topk, hidden, dtype=dtype)
        (dx,) = torch.autograd.grad(rows, x, g)
        want = torch.zeros(tokens, hidden, dtype=torch.float64, device="cuda").index_add_(0, at, g[:used].double())
        size = torch.zeros_like(want).index_add_(0, at, g[:used].double().abs())
        half = torch.finfo(dtype).eps / 2
        ref.check(dx, want, topk * UNIT * size * (1 + half) + half * want.abs(), (kind, "dx"))
        # The sort is linear: its differences are the sorted differences, to the bit where they are exact.
        d = torch.zeros_like(x)
        d[tokens // 2, hidden // 2] = 1.0
        moved = cuda_runtime.expert_sort(d, torch.from_numpy(ids).cuda(), experts)[0]
        change = float((moved.double() * g.double()).sum())
        assert abs(change - float(want[tokens // 2, hidden // 2])) <= 1e-9 * (1 + float(size.max()))


@pytest.mark.parametrize("how", ["all", "some", "none"])
@pytest.mark.parametrize("tokens,topk,experts,hidden", SIZES)
def test_return_and_its_gradients(cuda_runtime, tokens, topk, experts, hidden, how):
    ids = torch.from_numpy(_ids(tokens, tokens, topk, experts, how)).cuda()
    _, order = cuda_runtime.expert_sort(torch.zeros(tokens, 1, device="cuda"), ids, experts)
    inverse = order.inverse.long()
    has = inverse >= 0
    for kind, dtype in TYPES.items():
        for weight_type in (torch.float32, dtype, None):
            rows = _normal(3, tokens * topk, hidden, dtype=dtype).requires_grad_()
            residual = _normal(4, tokens, hidden, dtype=dtype).requires_grad_() if weight_type != dtype else None
            weights = None
            if weight_type is not None:
                weights = _normal(5, tokens, topk, dtype=weight_type).requires_grad_()
            out = cuda_runtime.expert_return(rows, order, weights, residual)
            taken = rows.detach().double()[inverse.clamp(min=0)] * has[..., None]
            w = weights.detach().double() if weights is not None else torch.ones(tokens, topk, device="cuda").double()
            res = residual.detach().double() if residual is not None else 0.0
            want = (w[..., None] * taken).sum(1) + res
            size = (w[..., None] * taken).abs().sum(1) + (res.abs() if residual is not None else 0.0)
            half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny * torch.finfo(dtype).eps
            ref.check(out, want, topk * UNIT * size * (1 + half) + half * want.abs() + tiny, (kind, "out"))
            g = _normal(6, tokens, hidden, dtype=dtype)
            needs = [t for t in (rows, weights, residual) if t is not None]
            grads = list(torch.autograd.grad(out, needs, g))
            gd = g.double()
            # drows: one product, rounded once.
            want = torch.zeros(tokens * topk + 1, hidden, dtype=torch.float64, device="cuda")
            want[torch.where(has, inverse, tokens * topk)] = w[..., None] * gd[:, None]
            want = want[:-1]
            ref.check(grads[0], want, (UNIT * (1 + half) + half) * want.abs() + tiny, (kind, "drows"))
            if weights is not None:
                # dweights: an FP32 sum of `hidden` products.
                want = (gd[:, None] * taken).sum(2)
                size = (gd[:, None] * taken).abs().sum(2)
                wh, wt = torch.finfo(weight_type).eps / 2, torch.finfo(weight_type).tiny
                ref.check(grads[1], want, hidden * UNIT * size * (1 + wh) + wh * want.abs() + wt, (kind, "dw"))
            if residual is not None:
                assert torch.equal(grads[-1], g)


def test_gradients_against_differences(cuda_runtime):
    """out is linear in the rows, the weights and the residual: <g, out(a + d) - out(a - d)> / 2 = <grad, d>."""
    tokens, topk, experts, hidden = 20, 4, 16, 48
    ids = torch.from_numpy(_ids(3, tokens, topk, experts, "some")).cuda()
    x = _normal(7, tokens, hidden).requires_grad_()
    rows, order = cuda_runtime.expert_sort(x, ids, experts)
    weights, residual = _normal(8, tokens, topk).requires_grad_(), _normal(9, tokens, hidden).requires_grad_()
    g = _normal(10, tokens, hidden)

    def value(x, weights, residual):
        r, o = cuda_runtime.expert_sort(x, ids, experts)
        return float((cuda_runtime.expert_return(r, o, weights, residual).double() * g.double()).sum())

    out = cuda_runtime.expert_return(rows, order, weights, residual)
    grads = torch.autograd.grad(out, (x, weights, residual), g)
    leaves = [t.detach() for t in (x, weights, residual)]
    for i, grad in enumerate(grads):
        d = _normal(11 + i, *leaves[i].shape)
        up, down = list(leaves), list(leaves)
        up[i], down[i] = leaves[i] + d, leaves[i] - d
        diff = (value(*up) - value(*down)) / 2
        want = float((grad.double() * d.double()).sum())
        # Every FP32 rounding of the two sides: (topk + 2) per value, and the sizes of the sums.
        size = sum(float(t.abs().max()) for t in leaves) ** 2 * float(g.abs().sum()) * (topk + 2)
        assert abs(diff - want) <= (topk + 4) * UNIT * 8 * size


@pytest.mark.parametrize("kind", list(TYPES))
def test_strides_types_and_addresses(cuda_runtime, kind):
    """Ids as the routing record holds them (row stride 9) and as int64, rows of x with a stride, off 16 bytes,
    repeated; an out with a stride; broadcast gradients."""
    dtype, tokens, topk, experts = TYPES[kind], 40, 8, 16
    record = torch.from_numpy(_ids(1, tokens, 9, experts, "all")).cuda()
    ids = record[:, :8]
    wide = _normal(20, tokens, 77, dtype=dtype)
    for hidden in (64, 33):
        for x in (wide[:, :hidden], wide[:, 3:3 + hidden], wide[:1, :hidden].expand(tokens, hidden),
                  wide[:, :hidden].t().contiguous().t()):
            rows, order = cuda_runtime.expert_sort(x, ids, experts)
            wide_rows, wide_order = cuda_runtime.expert_sort(x.contiguous(), ids.long().contiguous(), experts)
            assert torch.equal(rows, wide_rows) and torch.equal(order.inverse, wide_order.inverse)
            assert torch.equal(rows, x[(order.perm // topk).long()])
            weights = _normal(21, topk, tokens).t()
            buffer = torch.full((tokens, hidden + 5), 9.0, dtype=dtype, device="cuda")
            plain = cuda_runtime.expert_return(rows, order, weights, x)
            got = cuda_runtime.expert_return(rows, order, weights, x, out=buffer[:, 1:1 + hidden])
            assert torch.equal(got, plain)
            assert bool((buffer[:, 0] == 9).all()) and bool((buffer[:, 1 + hidden:] == 9).all())
    x = wide[:, :64].clone().requires_grad_()
    rows, order = cuda_runtime.expert_sort(x, ids, experts)
    cuda_runtime.expert_return(rows, order).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 8.0))


def test_empty_batches(cuda_runtime):
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    ids = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    rows, order = cuda_runtime.expert_sort(x, ids, 8)
    assert rows.shape == (0, 16) and not bool(order.offsets.any()) and order.offsets.shape == (9,)
    out = cuda_runtime.expert_return(rows, order, torch.zeros(0, 4, device="cuda", requires_grad=True))
    out.sum().backward()
    assert out.shape == (0, 16) and x.grad.shape == (0, 16)


def test_not_finite_rows_of_dropped_picks(cuda_runtime):
    """Rows that no pick reaches are not read: NaN there reaches neither the output nor a gradient."""
    ids = torch.tensor([[0, -1], [-1, 1]], dtype=torch.int32, device="cuda")
    _, order = cuda_runtime.expert_sort(torch.zeros(2, 8, device="cuda"), ids, 2)
    rows = torch.ones(4, 8, device="cuda")
    rows[2:] = float("nan")
    rows.requires_grad_()
    weights = torch.full((2, 2), 2.0, device="cuda", requires_grad=True)
    out = cuda_runtime.expert_return(rows, order, weights)
    assert torch.equal(out, torch.full((2, 8), 2.0, device="cuda"))
    drows, dw = torch.autograd.grad(out, (rows, weights), torch.ones_like(out))
    assert torch.equal(dw, torch.tensor([[8.0, 0.0], [0.0, 8.0]], device="cuda"))
    assert bool((drows[:2] == 2).all()) and not bool(drows[2:].any())


def test_rows_past_32_bit_offsets(cuda_runtime):
    """More than 2^31 elements of sorted rows."""
    tokens, topk, experts, hidden = 33000, 8, 16, 8200
    ids = torch.from_numpy(_ids(2, tokens, topk, experts, "all")).cuda()
    x = torch.randn(tokens, hidden, device="cuda").to(torch.bfloat16)
    rows, order = cuda_runtime.expert_sort(x, ids, experts)
    assert rows.numel() > 2 ** 31
    at = (order.perm // topk).long()
    for part in (slice(0, 3000), slice(-3000, None)):
        assert torch.equal(rows[part], x[at[part]])
    out = cuda_runtime.expert_return(rows, order, torch.full((tokens, topk), 0.125, device="cuda"))
    assert torch.equal(out, x)


@pytest.mark.parametrize("tokens", [300, 1500])  # a one-CTA sort, and a cluster's with a dependent launch
def test_streams_and_graphs(cuda_runtime, tokens):
    """On another stream, and a forward and backward pass captured and replayed on new values."""
    rt = cuda_runtime
    topk, experts, hidden = 4, 32, 64

    def step(x, ids, weights, g):
        rows, order = rt.expert_sort(x, ids, experts)
        out = rt.expert_return(rows, order, weights, x)
        return (out, *torch.autograd.grad(out, (x, weights), g))

    def inputs(seed):
        return (_normal(seed, tokens, hidden), torch.from_numpy(_ids(seed, tokens, topk, experts, "some")).cuda(),
                _normal(seed + 1, tokens, topk), _normal(seed + 2, tokens, hidden))

    first, second = inputs(30), inputs(40)
    for v in (first, second):
        v[0].requires_grad_()
        v[2].requires_grad_()
    want = [t.clone() for t in step(*second)]
    side = torch.cuda.Stream()
    rows, order = rt.expert_sort(second[0].detach(), second[1], experts, stream=side)
    out = rt.expert_return(rows, order, second[2].detach(), second[0].detach(), stream=side)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step(*first)
    with torch.no_grad():
        for a, b in zip(first, second):
            a.copy_(b)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_results_side_by_side_and_onto_the_residual(cuda_runtime):
    """The return into the columns beside its rows, and onto its residual: the bits of the plain call."""
    rt = cuda_runtime
    tokens, topk, experts, hidden = 70, 2, 6, 48
    ids = torch.from_numpy(_ids(60, tokens, topk, experts, "some")).cuda()
    rows, order = rt.expert_sort(_normal(61, tokens, hidden), ids, experts)
    w, residual = _normal(62, tokens, topk), _normal(63, tokens, hidden)
    want = rt.expert_return(rows, order, w, residual)
    both = torch.cat([rows, torch.full_like(rows, 3.0)], dim=1)
    out = rt.expert_return(both[:, :hidden], order, w, residual, out=both[:tokens, hidden:])
    assert torch.equal(out, want) and torch.equal(both[:, :hidden], rows) and bool((both[tokens:, hidden:] == 3).all())
    assert rt.expert_return(rows, order, w, residual, out=residual) is residual and torch.equal(residual, want)


def test_changed_order_is_seen_by_the_backward_pass(cuda_runtime):
    """The order is kept for the gradients: writing to it in between is an error, not another gradient."""
    x = _normal(64, 9, 8).requires_grad_()
    ids = torch.from_numpy(_ids(65, 9, 2, 4, "all")).cuda()
    rows, order = cuda_runtime.expert_sort(x, ids, 4)
    order.inverse.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        rows.sum().backward()


def test_refusals(cuda_runtime):
    rt = cuda_runtime
    x = torch.zeros(4, 8, device="cuda")
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    rows, order = rt.expert_sort(x, ids, 3)
    w = torch.ones(4, 2, device="cuda")
    bad = [
        lambda: rt.expert_sort(x.cpu(), ids, 3), lambda: rt.expert_sort(x.double(), ids, 3),
        lambda: rt.expert_sort(x[0], ids, 3), lambda: rt.expert_sort(x, ids.float(), 3),
        lambda: rt.expert_sort(x, ids[:3], 3), lambda: rt.expert_sort(x, ids.cpu(), 3),
        lambda: rt.expert_sort(x, ids, 0), lambda: rt.expert_sort(x, ids, 1025),
        lambda: rt.expert_sort(x, ids.repeat(1, 40), 3), lambda: rt.expert_sort(x, ids[:, :0], 3),
        lambda: rt.expert_sort(x[:, :0], ids, 3), lambda: rt.expert_return(rows[:7], order),
        lambda: rt.expert_return(rows.double(), order), lambda: rt.expert_return(rows, order, w.t()),
        lambda: rt.expert_return(rows, order, w.double()), lambda: rt.expert_return(rows, order, w.cpu()),
        lambda: rt.expert_return(rows, order, w, x[:3]), lambda: rt.expert_return(rows, order, w, x.half()),
        lambda: rt.expert_return(rows, order, w, out=x.half()),
        lambda: rt.expert_return(rows, order, w, out=x[:1].expand(4, 8)),
        lambda: rt.expert_return(rows, order, w.clone().requires_grad_(), out=x),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for out in (rows[2:6], rows[:4]):  # onto rows that are still to be read
        with pytest.raises(RuntimeError, match="overlap"):
            rt.expert_return(rows, order, w, out=out)
    wide = torch.zeros(5, 8, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        rt.expert_return(rows, order, w, wide[:4], out=wide[1:])
    # A gradient of a gradient is refused.
    y = x.clone().requires_grad_()
    r, _ = rt.expert_sort(y, ids, 3)
    (d,) = torch.autograd.grad(r, y, torch.ones_like(r).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    y = rows.clone().requires_grad_()
    r = rt.expert_return(y, order, w)
    (d,) = torch.autograd.grad(r, y, torch.ones_like(r).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


@pytest.mark.parametrize("tokens", [1, 5, 64, 300])
def test_run_of_a_layer(cuda_runtime, tokens):
    """Sort, gate and up product with SwiGLU, down product, weighted return onto the residual: the routed part of an
    NVFP4 layer with other routing than the bank's (top 3 of 12 with a dropped pick), against the formula in 64 bits."""
    rt, experts, topk, hidden, inner = cuda_runtime, 12, 3, 256, 96
    up = ref.random_matrix(experts, 2 * inner, hidden, 50)
    down = ref.random_matrix(experts, hidden, inner, 51)
    m_up, m_down = rt.upload_grouped(*(t.cuda() for t in up)), rt.upload_grouped(*(t.cuda() for t in down))
    x = _normal(52, tokens, hidden, dtype=torch.bfloat16)
    ids = torch.from_numpy(_ids(53, tokens, topk, experts, "some")).cuda()
    weights = torch.softmax(_normal(54, tokens, topk), dim=1)
    rows, order = rt.expert_sort(x, ids, experts)
    act = rt.linear_grouped(m_up, rows, order.offsets, activation="silu_mul")
    back = rt.linear_grouped(m_down, act, order.offsets)
    out = rt.expert_return(back, order, weights, x)
    want, tol = x.double(), torch.zeros(tokens, hidden, dtype=torch.float64, device="cuda")
    for t in range(tokens):
        for k in range(topk):
            e = int(ids[t, k])
            if e < 0:
                continue
            a, ea = ref.linear(x[t:t + 1], up[0][e].cuda(), up[1][e].cuda(), up[2][e].cuda(), None, "silu_mul")
            w = ref.weights(down[0][e].cuda(), down[1][e].cuda()) / down[2][e].double().cuda()
            b = a @ w.t()
            # The first product's error through the second, whose own sums and rounding are far below bf16's.
            eb = ea @ w.abs().t() + 2.0 ** -8 * b.abs() + 2.0 ** -16 * (a.abs() @ w.abs().t())
            want[t] += weights[t, k].double() * b[0]
            tol[t] += weights[t, k].double() * eb[0]
    ref.check(out, want, tol * 1.01 + 2.0 ** -8 * want.abs())
    m_up.close()
    m_down.close()
