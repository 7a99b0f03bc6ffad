"""Paths of the rotary, gated operators that only long inputs and large results
take: gradients over several tables of turns a workgroup, and results that go past
the caches. References are in 64 bits on the GPU."""

from __future__ import annotations

import pytest
import torch

import blocks_support as support
import cuvit_amd as cuvit
from test_gated_gpu import DEV, TYPES, operands
from test_qk_norm_gpu import Case
from test_rotary_gpu import positions_of

pytestmark = pytest.mark.gpu


def inside(produced, expected, bound):
    return bool(((produced.double() - expected).abs() <= bound).all())


# A workgroup's tokens, of which it holds the turns of 64 (32 pairs), of 8 (256
# pairs) and of 512 (4 pairs) at a time, or goes through 64 (none): each more than
# two times that, with a short last part and a short last workgroup.
LONG = [(13, 5101, 1, 1, 64, [16, 16]), (1, 9733, 1, 2, 512, [128, 128]), (7, 75001, 1, 1, 8, [2, 2]),
        (1, 70001, 2, 1, 24, []), (3, 35003, 1, 1, 72, [9, 9])]


class LongCase(Case):
    """With positions of each image's own."""

    def __init__(self, dtype, images, tokens, heads, kv_heads, head_dim, pairs, **more):
        super().__init__(dtype, images, tokens, heads, kv_heads, head_dim, pairs, **more)
        axes = max(len(pairs), 1)
        self.positions = positions_of(support.seeded(tokens), images, tokens, axes)
        self.problem.rotation.position_stride = tokens * axes


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("images,tokens,heads,kv_heads,head_dim,pairs", LONG)
def test_gradients_over_several_tables(dtype, layer, images, tokens, heads, kv_heads, head_dim, pairs):
    """The bounds are Case.check_backward's."""
    case = LongCase(dtype, images, tokens, heads, kv_heads, head_dim, pairs, layer=layer)
    out, sums = case.backward()
    case.qkv, case.grad, case.positions, case.frequencies = case.gpu(case.qkv, case.grad, case.positions,
                                                                     case.frequencies)
    case.gamma = case.gpu(*case.gamma)
    with torch.device(DEV):
        expected, size, d_gamma, size_gamma, d_beta, size_beta = support.qk_norm_gradients(
            case.qkv, case.grad, heads, kv_heads, layer, 1.0e-6, case.gamma, case.rotation())
    normed = heads + kv_heads
    bound = 2.0 ** -16.5 * size
    if dtype != torch.float32:
        bound = bound + support.ROUNDING[dtype] * expected.abs()
    assert inside(out[:, :, :normed], expected[:, :, :normed], bound[:, :, :normed])
    assert torch.equal(out[:, :, normed:], case.grad[:, :, normed:])
    unit = 2.0 ** -17 + (images * tokens * heads / 512 + 305) * support.ARITHMETIC
    assert inside(torch.stack(sums[:2]), d_gamma, unit * size_gamma)
    assert inside(torch.stack(sums[2:]), d_beta, unit * size_beta)


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("m,n,ldc,k", [(12608, 2048, 2048, 200), (12608, 1363, 1376, 72), (9232, 2048, 2056, 200),
                                       (9999, 1681, 1688, 64), (12608, 1363, 1363, 72)])
def test_large_products(m, n, ldc, k, keep):
    """More than 32 MB of C: whole 16-byte pieces of a row, a cut last one, room
    between the rows, and rows at any address."""
    dtype = torch.bfloat16
    assert m * n * 2 > 32 * 2 ** 20
    a, w, b = (t.to(DEV) for t in operands(dtype, m, n, k))
    problem = cuvit.gated_problem(m, n, k, cuvit.GATE_SILU)
    problem.ldc = ldc
    out = torch.full((m, ldc), 7.0, dtype=dtype, device=DEV)
    pre = torch.full((m, 2 * n), 7.0, dtype=dtype, device=DEV) if keep else None
    cuvit.gated_gemm(a, w, b, out, problem, preactivations=pre)
    expected, bound, z, error = support.gated(a, w, b, 0, dtype)
    assert inside(out[:, :n], expected, bound) and bool((out[:, n:] == 7.0).all())
    if keep:
        assert inside(pre, z, error)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,extra", [(4200, 1029, 0), (4200, 1032, 0), (4200, 1029, 11)])
def test_large_gradients_of_the_gate(dtype, m, n, extra):
    """More than 16 MB of gradients: rows at any address, whole pieces, room
    between the rows; and in the preactivations' place."""
    g = support.seeded(m + n)
    z = support.normal(g, m, 2 * n + extra, scale=2.0, dtype=dtype).to(DEV)
    d = support.normal(g, m, n + extra, dtype=dtype).to(DEV)
    assert m * 2 * n * z.element_size() > 16 * 2 ** 20
    problem = cuvit.gated_problem(m, n, 1, cuvit.GATE_SILU)
    problem.ldc, problem.ld_preactivations = n + extra, 2 * n + extra
    out = torch.full_like(z, 7.0)
    cuvit.gated_backward(z, d, out, problem)
    expected, bound = support.gated_gradient(z[:, :2 * n], d[:, :n], 0, dtype)
    assert inside(out[:, :2 * n], expected, bound) and bool((out[:, 2 * n:] == 7.0).all())
    room = z[:, 2 * n:].clone()
    cuvit.gated_backward(z, d, z, problem)
    assert torch.equal(z[:, :2 * n], out[:, :2 * n]) and torch.equal(z[:, 2 * n:], room)
