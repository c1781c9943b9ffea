"""The NVFP4 linear with its epilogue (Runtime.linear_fused) and its grouped form (Runtime.linear_grouped) against
their formulas in 64 bits (needs an sm_100a GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import fused_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _normal(seed, *shape, dtype=torch.float32, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()


def _matrix(rt, groups, rows, cols, seed, on_host=False):
    packed, scales, divisors = ref.random_matrix(groups, rows, cols, seed)
    if on_host:
        m = rt.upload_grouped(packed.numpy(), scales.numpy(), divisors.numpy())
    else:
        m = rt.upload_grouped(packed.cuda(), scales.cuda(), divisors.cuda())
    return m, packed.cuda(), scales.cuda(), divisors.cuda()


# vectors: one, the edges of the kernels' column tiles, and several tiles; cols: one block, odd numbers of blocks,
# not a multiple of a tile, several; rows: odd, below and across tiles.
SHAPES = [(1, 16, 16), (1, 128, 2048), (2, 33, 1040), (3, 1, 48), (8, 130, 272), (9, 257, 512), (17, 64, 80),
          (31, 200, 336), (32, 129, 1008), (33, 128, 256), (64, 300, 512), (65, 77, 144), (129, 260, 1008),
          (255, 128, 64), (257, 385, 528), (300, 1003, 1008)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vectors,rows,cols", SHAPES)
def test_shapes_and_types(cuda_runtime, kind, vectors, rows, cols):
    m, packed, scales, divisors = _matrix(cuda_runtime, 1, rows, cols, rows + cols)
    x = _normal(vectors + cols, vectors, cols, dtype=TYPES[kind])
    y = cuda_runtime.linear_fused(m, x)
    want, tol = ref.linear(x, packed[0], scales[0], divisors[0])
    assert y.dtype == x.dtype
    ref.check(y, want, tol)
    m.close()


@pytest.mark.parametrize("vectors", [1, 7, 40, 150])
@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu", "gelu_tanh", "relu_mul", "silu_mul", "gelu_mul",
                                        "gelu_tanh_mul"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_epilogues(cuda_runtime, kind, activation, vectors):
    rows, cols = 268, 400
    m, packed, scales, divisors = _matrix(cuda_runtime, 1, rows, cols, 5)
    width = rows // 2 if activation and activation.endswith("_mul") else rows
    dtype = TYPES[kind]
    x = _normal(1, vectors, cols, dtype=dtype)
    for bias_type in (dtype, torch.float32):
        bias = _normal(2, rows, dtype=bias_type)
        residual = _normal(3, vectors, width, dtype=dtype)
        y = cuda_runtime.linear_fused(m, x, bias=bias, activation=activation, residual=residual)
        want, tol = ref.linear(x, packed[0], scales[0], divisors[0], bias, activation, residual)
        ref.check(y, want, tol)
    # Onto the residual itself, and without bias or residual.
    z = cuda_runtime.linear_fused(m, x, bias=bias, activation=activation, residual=residual, out=residual)
    assert z is residual and torch.equal(z, y)
    y = cuda_runtime.linear_fused(m, x, activation=activation)
    want, tol = ref.linear(x, packed[0], scales[0], divisors[0], None, activation)
    ref.check(y, want, tol)
    m.close()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vectors", [5, 70])
def test_strides_and_shapes_of_tensors(cuda_runtime, kind, vectors):
    """Row strides, addresses off 16 bytes, leading axes, repeated rows, a transposed x; what lies around out stays."""
    rows, cols, dtype = 150, 96, TYPES[kind]
    m, packed, scales, divisors = _matrix(cuda_runtime, 1, rows, cols, 6)
    wide = _normal(4, vectors, cols + 13, dtype=dtype)
    for x in (wide[:, :cols], wide[:, 5:5 + cols], wide[:1, 8:8 + cols].expand(vectors, cols),
              wide[:, :cols].t().contiguous().t()):
        want, tol = ref.linear(x, packed[0], scales[0], divisors[0])
        buffer = torch.full((vectors, rows + 9), 7.0, dtype=dtype, device="cuda")
        got = cuda_runtime.linear_fused(m, x, out=buffer[:, 3:3 + rows])
        ref.check(got, want, tol)
        assert bool((buffer[:, :3] == 7).all()) and bool((buffer[:, 3 + rows:] == 7).all())
        res = buffer[:, 3:3 + rows].clone()
        want, tol = ref.linear(x, packed[0], scales[0], divisors[0], residual=res)
        ref.check(cuda_runtime.linear_fused(m, x, residual=buffer[:, 3:3 + rows]), want, tol)
    x = wide[:, :cols]
    want, tol = ref.linear(x, packed[0], scales[0], divisors[0])
    ref.check(cuda_runtime.linear_fused(m, x.reshape(1, vectors, 1, cols)).reshape(vectors, rows), want, tol)
    assert cuda_runtime.linear_fused(m, x[0]).shape == (rows,)
    assert cuda_runtime.linear_fused(m, x[:0]).shape == (0, rows)
    m.close()


@pytest.mark.parametrize("vectors", [4, 50])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_ranges_of_values(cuda_runtime, kind, vectors):
    """Rows of zeros, of tiny and of huge values, an outlier beside small values, and values that are not finite in
    some rows only: they stay in their rows."""
    rows, cols, dtype = 64, 256, TYPES[kind]
    m, packed, scales, divisors = _matrix(cuda_runtime, 1, rows, cols, 7)
    x = _normal(9, vectors, cols)
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e30
    x[3, 7] = 3e6
    x = x.to(dtype)
    want, tol = ref.linear(x, packed[0], scales[0], divisors[0])
    ref.check(cuda_runtime.linear_fused(m, x), want, tol)
    clean = cuda_runtime.linear_fused(m, x)
    y = x.clone()
    y[1, 3], y[2, 100], y[2, 101] = float("inf"), float("nan"), float("-inf")
    got = cuda_runtime.linear_fused(m, y)
    keep = [i for i in range(vectors) if i not in (1, 2)]
    assert torch.equal(got[keep], clean[keep])
    assert bool(got[2].isnan().all())
    w = ref.weights(packed, scales)[0, :, 3]
    assert bool((got[1] == torch.where(w > 0, float("inf"), float("-inf")).to(dtype))[w != 0].all())
    assert bool(got[1].isnan()[w == 0].all())  # zero times infinity
    m.close()


def test_matrix_of_the_dense_upload(cuda_runtime):
    """A matrix uploaded for the FP32 linear works here too; a grouped upload is refused there."""
    packed, scales, divisors = ref.random_matrix(1, 96, 320, 8)
    m = cuda_runtime.upload(packed[0].numpy(), scales[0].numpy(), float(divisors[0]))
    for vectors in (1, 3, 50):
        x = _normal(10, vectors, 320)
        want, tol = ref.linear(x, packed[0].cuda(), scales[0].cuda(), divisors[0].cuda())
        ref.check(cuda_runtime.linear_fused(m, x), want, tol)
    g = cuda_runtime.upload_grouped(packed.numpy(), scales.numpy(), divisors.numpy())
    with pytest.raises(RuntimeError, match="linear_fused"):
        cuda_runtime.linear_tensor(g, x)
    with pytest.raises(RuntimeError, match="linear_fused"):
        cuda_runtime.linear(g, x.cpu().numpy())
    m.close()
    g.close()


def test_long_rows(cuda_runtime):
    """The most columns the upload takes, one row of x and several."""
    rows, cols = 40, 49152
    m, packed, scales, divisors = _matrix(cuda_runtime, 1, rows, cols, 9)
    for kind in TYPES:
        for vectors in (1, 3, 40):
            x = _normal(11, vectors, cols, dtype=TYPES[kind])
            want, tol = ref.linear(x, packed[0], scales[0], divisors[0])
            ref.check(cuda_runtime.linear_fused(m, x), want, tol, (kind, vectors))
    m.close()


# ------------------------------------------------------------------ groups


def _check_grouped(rt, m, packed, scales, divisors, x, offsets, bias=None, activation=None):
    o = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y = rt.linear_grouped(m, x, o, bias=bias, activation=activation)
    width = y.shape[1]
    for g in range(len(offsets) - 1):
        a, b = offsets[g], offsets[g + 1]
        if a < b:
            want, tol = ref.linear(x[a:b], packed[g], scales[g], divisors[g], None if bias is None else bias[g],
                                   activation)
            ref.check(y[a:b], want, tol, g)
    assert not bool(y[:offsets[0]].any()) and not bool(y[offsets[-1]:].any())
    given = torch.full((x.shape[0], width + 3), 5.0, dtype=x.dtype, device="cuda")
    got = rt.linear_grouped(m, x, o, bias=bias, activation=activation, out=given[:, 1:1 + width])
    assert torch.equal(got[offsets[0]:offsets[-1]], y[offsets[0]:offsets[-1]])
    assert bool((given[:offsets[0]] == 5).all()) and bool((given[offsets[-1]:] == 5).all())
    assert bool((given[:, 0] == 5).all()) and bool((given[:, 1 + width:] == 5).all())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("offsets", [
    [0, 1, 1, 1, 1], [0, 0, 0, 0, 0], [0, 1, 2, 3, 4], [0, 5, 5, 38, 40], [2, 2, 9, 9, 12], [0, 64, 65, 200, 333],
    [0, 0, 0, 0, 300], [0, 130, 130, 387, 500]])
def test_groups(cuda_runtime, kind, offsets):
    rows, cols = 134, 144
    m, packed, scales, divisors = _matrix(cuda_runtime, 4, rows, cols, 12, on_host=True)
    x = _normal(13, offsets[-1] + 3, cols, dtype=TYPES[kind])
    bias = _normal(14, 4, rows, dtype=TYPES[kind])
    for activation in (None, "silu_mul"):
        _check_grouped(cuda_runtime, m, packed, scales, divisors, x, offsets, bias, activation)
    _check_grouped(cuda_runtime, m, packed, scales, divisors, x, offsets)
    m.close()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("offsets", [[0, 2], [0, 4], [1, 10], [0, 0, 17], [0, 31, 33], [3, 3, 3, 70]])
def test_few_groups_of_few_rows(cuda_runtime, kind, offsets):
    """Fewer rows than a tile of the many-row kernel loads, and ranges that end off its tiles."""
    m, packed, scales, divisors = _matrix(cuda_runtime, len(offsets) - 1, 72, 208, 31)
    x = _normal(32, offsets[-1] + 1, 208, dtype=TYPES[kind])
    _check_grouped(cuda_runtime, m, packed, scales, divisors, x, offsets, activation="silu_mul")
    m.close()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("offsets", [[0, 1, 2, 3, 4, 5, 6], [2, 2, 8, 9, 9, 14, 15], [0, 8, 16, 16, 17, 18, 18],
                                     [0, 3, 2, 5, 4, 9, 9], [0, 9, 10, 11, 11, 11, 12], [0, 0, 0, 0, 0, 0, 16]])
def test_rows_of_several_groups_staged_together(cuda_runtime, kind, offsets):
    """Few rows over groups of few weight rows: a block's tiles cross groups that are empty, full or too large to share
    its stage. Offsets that decrease give some row to two groups, and the rows of neither are compared."""
    m, packed, scales, divisors = _matrix(cuda_runtime, 6, 40, 272, 33)
    x = _normal(34, 18, 272, dtype=TYPES[kind])
    if all(a <= b for a, b in zip(offsets, offsets[1:])):
        bias = _normal(35, 6, 40, dtype=TYPES[kind])
        _check_grouped(cuda_runtime, m, packed, scales, divisors, x, offsets, bias=bias, activation="relu")
    else:
        y = cuda_runtime.linear_grouped(m, x, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        owners = [[g for g in range(6) if offsets[g] <= v < offsets[g + 1]] for v in range(18)]
        for v, own in enumerate(owners):
            if len(own) == 1:
                want, tol = ref.linear(x[v:v + 1], packed[own[0]], scales[own[0]], divisors[own[0]])
                ref.check(y[v:v + 1], want, tol, v)
    m.close()


@pytest.mark.parametrize("groups,most", [(1, 50), (37, 9), (300, 3), (1024, 2), (16, 200)])
def test_many_groups_of_uneven_sizes(cuda_runtime, groups, most):
    rows, cols = 80, 64
    m, packed, scales, divisors = _matrix(cuda_runtime, groups, rows, cols, 15)
    counts = np.random.default_rng(groups).integers(0, most + 1, groups)
    offsets = [0, *np.cumsum(counts).tolist()]
    x = _normal(16, max(1, offsets[-1]), cols, dtype=torch.bfloat16)
    _check_grouped(cuda_runtime, m, packed, scales, divisors, x, offsets, None, "gelu_tanh")
    m.close()


def test_offsets_outside_the_rows_are_kept_inside(cuda_runtime):
    """Numbers that no sort writes (below zero, past the rows, decreasing) read and write inside the call's rows."""
    m, packed, scales, divisors = _matrix(cuda_runtime, 4, 64, 64, 17)
    for vectors in (20, 200):
        x = _normal(18, vectors, 64, dtype=torch.float16)
        guard = torch.full((3 * vectors, 64), 3.0, dtype=torch.float16, device="cuda")
        out = guard[vectors:2 * vectors]
        o = torch.tensor([-5, 9, 4, vectors + 1000, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
        cuda_runtime.linear_grouped(m, x, o, out=out)
        torch.cuda.synchronize()
        assert bool((guard[:vectors] == 3).all()) and bool((guard[2 * vectors:] == 3).all())
    m.close()


# ------------------------------------------------------------------ streams, graphs, refusals


def test_streams_graphs_and_calls_at_once(cuda_runtime):
    """Two streams on one matrix at once, an explicit stream, and two captured calls replayed on new inputs: the bits
    of the plain call each time."""
    rows, cols = 200, 512
    m, packed, scales, divisors = _matrix(cuda_runtime, 1, rows, cols, 19)
    for dtype in (torch.bfloat16, torch.float32):
        for vectors in (2, 100):
            xs = [_normal(20 + i, vectors, cols, dtype=dtype) for i in range(4)]
            plain = [cuda_runtime.linear_fused(m, x, activation="silu") for x in xs]
            torch.cuda.synchronize()
            streams = [torch.cuda.Stream() for _ in xs]
            got = [cuda_runtime.linear_fused(m, x, activation="silu", stream=s) for x, s in zip(xs, streams)]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, plain))
            graphs, inputs, outputs = [], [], []
            for i in range(2):
                inputs.append(xs[i].clone())
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    outputs.append(cuda_runtime.linear_fused(m, inputs[i], activation="silu"))
                graphs.append(g)
            for i in range(2):
                inputs[i].copy_(xs[2 + i])
            torch.cuda.synchronize()
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(outputs[i], plain[2 + i]) for i in range(2))
    m.close()
    cuda_runtime.synchronize()


def test_grouped_streams_graphs_and_calls_at_once(cuda_runtime):
    """The grouped form on two streams at once, and two captured calls replayed together on new rows and offsets."""
    groups, rows, cols = 6, 136, 256
    m, *_ = _matrix(cuda_runtime, groups, rows, cols, 24)
    for dtype in (torch.float16, torch.float32):
        for cuts in (([0, 1, 1, 3, 4, 4, 6], [0, 2, 2, 2, 3, 6, 6]), ([0, 90, 91, 150, 300, 300, 400],
                                                                      [0, 0, 0, 399, 400, 400, 400])):
            xs = [_normal(25 + i, cuts[0][-1], cols, dtype=dtype) for i in range(2)]
            os = [torch.tensor(c, dtype=torch.int32, device="cuda") for c in cuts]
            plain = [[cuda_runtime.linear_grouped(m, x, o, activation="gelu_mul") for o in os] for x in xs]
            torch.cuda.synchronize()
            streams = [torch.cuda.Stream() for _ in xs]
            got = [cuda_runtime.linear_grouped(m, x, o, activation="gelu_mul", stream=s)
                   for x, o, s in zip(xs, os, streams)]
            torch.cuda.synchronize()
            assert torch.equal(got[0], plain[0][0]) and torch.equal(got[1], plain[1][1])
            graphs, inputs, outputs = [], [], []
            for i in range(2):
                inputs.append((xs[i].clone(), os[i].clone()))
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    outputs.append(cuda_runtime.linear_grouped(m, *inputs[i], activation="gelu_mul"))
                graphs.append(g)
            for i in range(2):
                inputs[i][0].copy_(xs[1 - i])
                inputs[i][1].copy_(os[1 - i])
            torch.cuda.synchronize()
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outputs[0], plain[1][1]) and torch.equal(outputs[1], plain[0][0])
    m.close()
    cuda_runtime.synchronize()


@pytest.mark.parametrize("vectors", [1, 6, 40])
def test_results_in_the_memory_of_the_inputs(cuda_runtime, vectors):
    """Into the columns beside x (the bits of the plain call); onto x, or across the residual's rows, is refused."""
    rt, cols = cuda_runtime, 64
    m, *_ = _matrix(rt, 1, 64, cols, 27)
    for dtype in TYPES.values():
        both = _normal(28, vectors + 1, 2 * cols, dtype=dtype)
        x, beside = both[:vectors, :cols], both[:vectors, cols:]
        want = rt.linear_fused(m, x, activation="relu", residual=beside)
        with pytest.raises(RuntimeError, match="overlap"):
            rt.linear_fused(m, x, out=x)
        with pytest.raises(RuntimeError, match="overlap"):
            rt.linear_fused(m, x, out=both[:vectors, cols // 2:cols // 2 + cols])
        if vectors > 1:
            with pytest.raises(RuntimeError, match="overlap"):
                rt.linear_fused(m, x.clone(), residual=beside, out=both[1:, cols:])
        assert torch.equal(rt.linear_fused(m, x, activation="relu", residual=beside, out=beside), want)
    g, *_ = _matrix(rt, 2, 64, cols, 29)
    x = _normal(30, 3, cols)
    with pytest.raises(RuntimeError, match="overlap"):
        rt.linear_grouped(g, x, torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"), out=x)
    m.close()
    g.close()


def test_refusals(cuda_runtime):
    rt = cuda_runtime
    m, *_ = _matrix(rt, 1, 65, 64, 21)
    g, *_ = _matrix(rt, 2, 64, 64, 22)
    x = _normal(23, 3, 64, dtype=torch.bfloat16)
    o = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    bad = [
        lambda: rt.linear_fused(m, x.cpu()), lambda: rt.linear_fused(m, x.double()), lambda: rt.linear_fused(m, x[:, :48]),
        lambda: rt.linear_fused(m, x, activation="tanh"), lambda: rt.linear_fused(m, x, activation="silu_mul"),
        lambda: rt.linear_fused(g, x), lambda: rt.linear_fused(m, x, bias=x[0]),
        lambda: rt.linear_fused(m, x, bias=torch.zeros(65)), lambda: rt.linear_fused(m, x, residual=x),
        lambda: rt.linear_fused(m, x, residual=torch.zeros(3, 65, device="cuda")),
        lambda: rt.linear_fused(m, x, out=torch.empty(65, 3, dtype=x.dtype, device="cuda").t()),
        lambda: rt.linear_fused(m, x, out=torch.empty(1, 65, dtype=x.dtype, device="cuda").expand(3, 65)),
        lambda: rt.linear_fused(m, x.float().requires_grad_()),
        lambda: rt.linear_grouped(g, x, o.long()), lambda: rt.linear_grouped(g, x, o[:2]),
        lambda: rt.linear_grouped(g, x, o.cpu()), lambda: rt.linear_grouped(g, x[None], o),
        lambda: rt.linear_grouped(g, x, o, bias=x[0]),
        lambda: rt.upload_grouped(torch.zeros(2, 3, 4), torch.zeros(2, 3, 1), torch.ones(2)),
        lambda: rt.upload_grouped(np.zeros((2, 3, 8), np.uint8), np.zeros((2, 3, 1), np.uint8), np.ones(3, np.float32)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for shape in ((2, 3, 4), (2, 3, 24577)):  # 8 columns; more than the upload takes
        with pytest.raises(RuntimeError, match=r"failed \(1\)"):
            rt.upload_grouped(np.zeros(shape, np.uint8), np.zeros((2, 3, max(1, shape[2] // 8)), np.uint8),
                              np.ones(2, np.float32))
    with torch.no_grad():
        assert not rt.linear_fused(m, x.float().requires_grad_()).requires_grad
    # At the C ABI: a workspace that is missing, too small or off its alignment, before anything is enqueued.
    y = torch.empty(40, 65, device="cuda")
    v = _normal(24, 40, 64)
    size = rt.lib.nvfp4_linear_workspace_bytes(m.handle, v.data_ptr(), 2, 64, 40, 0)
    space = torch.empty(size + 256, dtype=torch.uint8, device="cuda")
    for at, given in ((None, size), (space.data_ptr(), size - 1), (space.data_ptr() + 16, size)):
        assert rt.lib.nvfp4_linear_fused(rt.handle, m.handle, v.data_ptr(), 2, 64, 40, None, 0, 0, None, 0, y.data_ptr(),
                                         65, at, given, None) == 1
    m.close()
    g.close()
