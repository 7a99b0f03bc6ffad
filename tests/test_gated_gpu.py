"""The gated product and its gate's gradient against 64 bits."""

from __future__ import annotations

import pytest
import torch

import blocks_support as support
import cuvit_amd as cuvit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16]


def operands(dtype, m, n, k, bias=True, seed=0):
    g = support.seeded(seed + m + 3 * n + 7 * k)
    a = support.normal(g, m, k, dtype=dtype)
    w = support.normal(g, 2 * n, k, scale=max(k, 1) ** -0.5, dtype=dtype)
    return a, w, support.normal(g, 2 * n, scale=0.5) if bias else None


def check(dtype, m, n, k, kind=cuvit.GATE_SILU, bias=True, keep=False, seed=0):
    a, w, b = operands(dtype, m, n, k, bias, seed)
    out = torch.full((m, n), 7.0, dtype=dtype, device=DEV)
    pre = torch.full((m, 2 * n), 7.0, dtype=dtype, device=DEV) if keep else None
    cuvit.gated_gemm(a.to(DEV), w.to(DEV), None if b is None else b.to(DEV), out, cuvit.gated_problem(m, n, k, kind),
                     preactivations=pre)
    expected, bound, z, error = support.gated(a, w, b, kind, dtype)
    assert support.worst(out, expected, bound) <= 1.0
    if keep:
        assert support.worst(pre, z, error) <= 1.0
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_activations(dtype, kind, keep, bias):
    check(dtype, 70, 72, 64, kind, bias, keep)
    check(dtype, 3, 40, 136, kind, bias, keep)
    check(dtype, 33, 19, 77, kind, bias, keep)


# One problem for each tile and more of its kind: rows and columns of tiles that
# are cut, several to an XCD (test_gated_choice_cpu.py checks that they reach it).
TILES = [("64x32 alone", 100, 150, 136), ("64x64 alone", 394, 2048, 768), ("64x64", 700, 1501, 264),
         ("128x64", 1576, 2048, 768), ("192x128", 2308, 2048, 768), ("192x128", 4616, 1001, 72),
         ("256x128", 3152, 2048, 768), ("320x128", 4616, 2048, 768), ("320x128", 9232, 1001, 72)]
TILES_F32 = [("32x16 alone", 100, 150, 132), ("32x32 alone", 200, 1001, 132), ("32x32", 788, 1365, 100),
             ("64x32", 3152, 2048, 260)]


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("dtype,name,m,n,k", [(torch.bfloat16, *t) for t in TILES] + [(torch.float32, *t) for t in TILES_F32])
def test_each_tile(dtype, name, m, n, k, keep):
    """Against 64 bits on the GPU, and twice the same bits."""
    a, w, b = (t.to(DEV) for t in operands(dtype, m, n, k))
    problem = cuvit.gated_problem(m, n, k, cuvit.GATE_SILU)
    results = []
    for _ in range(2):
        out = torch.full((m, n), 7.0, dtype=dtype, device=DEV)
        pre = torch.full((m, 2 * n), 7.0, dtype=dtype, device=DEV) if keep else None
        cuvit.gated_gemm(a, w, b, out, problem, preactivations=pre)
        results.append((out, pre))
    expected, bound, z, error = (t.cpu() for t in support.gated(a, w, b, 0, dtype))
    assert support.worst(results[0][0], expected, bound) <= 1.0
    assert torch.equal(results[0][0], results[1][0])
    if keep:
        assert support.worst(results[0][1], z, error) <= 1.0 and torch.equal(results[0][1], results[1][1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 2, 7, 15, 16, 17, 31, 33, 63, 64, 65, 130, 197])
@pytest.mark.parametrize("n,k", [(64, 192), (65, 64), (200, 100), (17, 513)])
def test_rows(dtype, m, n, k):
    check(dtype, m, n, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 16, 90])
@pytest.mark.parametrize("n", [1, 3, 4, 15, 31, 33, 63, 127, 129, 256, 341])
def test_columns(dtype, m, n):
    check(dtype, m, n, 96, keep=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 5, 66])
@pytest.mark.parametrize("k", [1, 2, 7, 8, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 130, 257, 512, 1000, 1024, 2056])
def test_depths(dtype, m, k):
    check(dtype, m, 48, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1576, 512, 192), (788, 1024, 384), (3152, 2048, 768), (12608, 512, 192),
                                   (577, 1365, 512), (2000, 130, 770), (1, 2048, 768), (4, 2048, 768), (16, 8192, 1024),
                                   (300, 2048, 2048)])
def test_layers(dtype, m, n, k):
    """Layers' sizes against 64 bits on the GPU."""
    a, w, b = (t.to(DEV) for t in operands(dtype, m, n, k))
    out = torch.empty(m, n, dtype=dtype, device=DEV)
    pre = torch.empty(m, 2 * n, dtype=dtype, device=DEV)
    cuvit.gated_gemm(a, w, b, out, cuvit.gated_problem(m, n, k, cuvit.GATE_GELU), preactivations=pre)
    expected, bound, z, error = (t.cpu() for t in support.gated(a, w, b, 1, dtype))
    assert support.worst(out, expected, bound) <= 1.0 and support.worst(pre, z, error) <= 1.0


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(65, 31, 33), (100, 1365, 513), (394, 683, 257), (788, 1365, 77), (3152, 1365, 131),
                                   (2100, 2048, 63)])
def test_tiles_of_loose_rows(dtype, m, n, k, keep):
    """Rows that are no whole 16-byte chunks, from a few tiles to several a CU:
    against 64 bits on the GPU, and twice the same bits."""
    a, w, b = (t.to(DEV) for t in operands(dtype, m, n, k))
    results = []
    for _ in range(2):
        out = torch.full((m, n), 7.0, dtype=dtype, device=DEV)
        pre = torch.full((m, 2 * n), 7.0, dtype=dtype, device=DEV) if keep else None
        cuvit.gated_gemm(a, w, b, out, cuvit.gated_problem(m, n, k), preactivations=pre)
        results.append((out, pre))
    expected, bound, z, error = (t.cpu() for t in support.gated(a, w, b, 0, dtype))
    assert support.worst(results[0][0], expected, bound) <= 1.0 and torch.equal(results[0][0], results[1][0])
    if keep:
        assert support.worst(results[0][1], z, error) <= 1.0 and torch.equal(results[0][1], results[1][1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 9, 16, 17, 100])
@pytest.mark.parametrize("n,k,extra", [(72, 64, 8), (72, 64, 1), (33, 50, 3), (128, 128, 4)])
def test_leading_dimensions_and_neighbours(dtype, m, n, k, extra):
    """Rows apart give the packed rows' bits, or another kernel's within the
    bound; what lies between them stays. NaN behind A's and B's rows is not read
    into a sum."""
    a, w, b = operands(dtype, m, n, k)
    problem = cuvit.gated_problem(m, n, k, cuvit.GATE_SILU)
    problem.lda = problem.ldb = k + extra
    problem.ldc, problem.ld_preactivations = n + extra, 2 * n + extra

    def padded(t, fill):
        wide = torch.full((t.shape[0], t.shape[1] + extra), fill, dtype=t.dtype)
        wide[:, :t.shape[1]] = t
        return wide.to(DEV)

    nan = float("nan")
    out = torch.full((m, n + extra), 7.0, dtype=dtype, device=DEV)
    pre = torch.full((m, 2 * n + extra), 7.0, dtype=dtype, device=DEV)
    cuvit.gated_gemm(padded(a, nan), padded(w, nan), b.to(DEV), out, problem, preactivations=pre)
    expected, bound, z, error = support.gated(a, w, b, 0, dtype)
    assert support.worst(out[:, :n], expected, bound) <= 1.0 and support.worst(pre[:, :2 * n], z, error) <= 1.0
    assert bool((out[:, n:] == 7.0).all()) and bool((pre[:, 2 * n:] == 7.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 16, 70])
def test_any_address(dtype, m):
    """Operands off a 16-byte address, each by itself and all together."""
    n, k = 72, 64
    a, w, b = operands(dtype, m, n, k)
    expected, bound, _, _ = support.gated(a, w, b, 0, dtype)

    def at(t, shift):
        room = torch.full((t.numel() + 16,), 7.0, dtype=t.dtype, device=DEV)
        room[shift:shift + t.numel()] = t.flatten().to(DEV)
        return room, room[shift:shift + t.numel()]

    for shifts in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (2, 4, 3, 5)):
        room, out = at(torch.full((m, n), 7.0, dtype=dtype), shifts[3])
        cuvit.gated_gemm(at(a, shifts[0])[1], at(w, shifts[1])[1], at(b, shifts[2])[1], out,
                         cuvit.gated_problem(m, n, k))
        assert support.worst(out.reshape(m, n), expected, bound) <= 1.0
        assert bool((room[:shifts[3]] == 7.0).all()) and bool((room[shifts[3] + m * n:] == 7.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 20])
def test_no_depth_is_the_bias(dtype, m):
    bias = support.normal(support.seeded(1), 20)
    out = torch.full((m, 10), 7.0, dtype=dtype, device=DEV)
    some = torch.zeros(1, dtype=dtype, device=DEV)
    cuvit.gated_gemm(some, some, bias.to(DEV), out, cuvit.gated_problem(m, 10, 0, cuvit.GATE_SILU))
    expected = (support.activation(0, bias[:10].double()) * bias[10:].double()).expand(m, -1)
    assert support.worst(out, expected, support.ROUNDING[dtype] * expected.abs() + 2.0 ** -20) <= 1.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [2, 50])
def test_infinities_and_nan_stay_in_their_rows(dtype, m):
    n, k = 64, 128
    a, w, b = (t.to(DEV) for t in operands(dtype, m, n, k))
    clean, spoiled = (torch.empty(m, n, dtype=dtype, device=DEV) for _ in range(2))
    cuvit.gated_gemm(a, w, b, clean, cuvit.gated_problem(m, n, k))
    a[1, 3] = float("nan")
    w[5] = float("inf")
    cuvit.gated_gemm(a, w, b, spoiled, cuvit.gated_problem(m, n, k))
    rows, columns = [r for r in range(m) if r != 1], [c for c in range(n) if c != 5]
    assert torch.equal(spoiled[rows][:, columns], clean[rows][:, columns])
    assert bool(torch.isnan(spoiled[1]).all()) and not bool(torch.isfinite(spoiled[0, 5]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_ends_of_the_activations(dtype, kind):
    """Gates far below and above zero: 0 (or its sign) and the gate itself."""
    bias = torch.tensor([-1e4, -200.0, -88.0, -40.0, -9.0, 0.0, 9.0, 40.0, 88.0, 200.0, 1e4] + [1.0] * 11)
    for m in (1, 20):
        out = torch.full((m, 11), 7.0, dtype=dtype, device=DEV)
        zero = torch.zeros(m, 8, dtype=dtype, device=DEV)
        cuvit.gated_gemm(zero, torch.zeros(22, 8, dtype=dtype, device=DEV), bias.to(DEV), out,
                         cuvit.gated_problem(m, 11, 8, kind))
        expected = support.activation(kind, bias[:11].double()).expand(m, -1)
        assert support.worst(out, expected, support.ROUNDING[dtype] * expected.abs() + 2.0 ** -20) <= 1.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 8), (3, 7), (5, 64), (70, 33), (197, 683), (130, 129), (2000, 8)])
def test_gradient(dtype, kind, m, n):
    g = support.seeded(m + n)
    z, d = support.normal(g, m, 2 * n, scale=2.0, dtype=dtype), support.normal(g, m, n, dtype=dtype)
    out = torch.full((m, 2 * n), 7.0, dtype=dtype, device=DEV)
    problem = cuvit.gated_problem(m, n, 1, kind)
    there = z.to(DEV)
    cuvit.gated_backward(there, d.to(DEV), out, problem)
    expected, bound = support.gated_gradient(z, d, kind, dtype)
    assert support.worst(out, expected, bound) <= 1.0
    cuvit.gated_backward(there, d.to(DEV), there, problem)  # in their place
    assert torch.equal(there, out)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_rows_apart_and_far_gates(dtype):
    g = support.seeded(12)
    m, n, extra = 9, 21, 5
    z, d = support.normal(g, m, 2 * n, scale=30.0, dtype=dtype), support.normal(g, m, n, dtype=dtype)
    for kind in range(3):
        problem = cuvit.gated_problem(m, n, 1, kind)
        problem.ldc, problem.ld_preactivations = n + extra, 2 * n + extra
        pre = torch.full((m, 2 * n + extra), float("nan"), dtype=dtype)
        pre[:, :2 * n] = z
        grad = torch.full((m, n + extra), float("nan"), dtype=dtype)
        grad[:, :n] = d
        out = torch.full((m, 2 * n + extra), 7.0, dtype=dtype, device=DEV)
        cuvit.gated_backward(pre.to(DEV), grad.to(DEV), out, problem)
        expected, bound = support.gated_gradient(z, d, kind, dtype)
        assert support.worst(out[:, :2 * n], expected, bound) <= 1.0
        assert bool((out[:, 2 * n:] == 7.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_gradient_of_gates_whose_squares_overflow(dtype, kind):
    """Slopes of 0 and 1, activations of 0 and the gate: exact, as d and value are 1."""
    gate = torch.tensor([1e15, 1.8e19, 1e20, 3e38], dtype=dtype)
    gate = torch.cat([-gate, gate, gate.new_zeros(3)])  # 11: a whole run and a cut one
    z = torch.cat([gate, torch.ones_like(gate)]).to(DEV)
    out = torch.full_like(z, 7.0)
    cuvit.gated_backward(z, torch.ones_like(gate).to(DEV), out, cuvit.gated_problem(1, 11, 1, kind))
    slopes = torch.tensor([0.0] * 4 + [1.0] * 4 + [0.5] * 3, dtype=dtype)
    assert torch.equal(out[:11].cpu(), slopes)
    assert torch.equal(out[11:].cpu(), gate.clamp(min=0))


def test_refused_tensors():
    a, w, b = (t.to(DEV) for t in operands(torch.float32, 4, 6, 8))
    out = torch.full((4, 6), 7.0, device=DEV)
    problem = cuvit.gated_problem(4, 6, 8)
    for arguments, more, message in [
            ((a[:3], w, b, out), {}, "A holds 24 elements"), ((a, w[:11], b, out), {}, "B holds 88"),
            ((a, w, b[:11], out), {}, "bias holds 11"), ((a, w, b, out[:3]), {}, "C holds 18"),
            ((a, w, b, out), {"preactivations": out}, "preactivations holds 24"),
            ((a, w.bfloat16(), b, out), {}, "B holds torch.bfloat16"), ((a.t().contiguous().t(), w, b, out), {},
                                                                       "A is not contiguous")]:
        with pytest.raises(cuvit.InvalidArgument, match=message):
            cuvit.gated_gemm(*arguments, problem, **more)
    pre = torch.zeros(4, 12, device=DEV)
    with pytest.raises(cuvit.InvalidArgument, match="grad holds 18"):
        cuvit.gated_backward(pre, out[:3], pre, problem)
    with pytest.raises(cuvit.InvalidArgument, match="grad_preactivations holds 24"):
        cuvit.gated_backward(pre, out, out.clone(), problem)
    assert bool((out == 7.0).all())
