"""Rotations and norms of 2^31 - 2 tokens, one less than a call may have: every
image as if it were the only one; and strides that no tensor holds."""

from __future__ import annotations

import pytest
import torch

import blocks_support as support
import cuvit_amd as cuvit
from test_rotary_gpu import ladder, positions_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
IMAGES, TOKENS = 42966, 49981
assert IMAGES * TOKENS == 2 ** 31 - 2


def images_are(x, alone):
    """Whether each of x's images has the bits of @p alone."""
    return all(bool((part.view(torch.int16) == alone.view(torch.int16)).all()) for part in x.split(2048))


def test_rotary():
    g = support.seeded(1)
    one = support.normal(g, 1, TOKENS, 1, 2, dtype=torch.bfloat16).to(DEV)
    at, turns = positions_of(g, TOKENS, 1).to(DEV), ladder([1]).to(DEV)
    x = one.repeat(IMAGES, 1, 1, 1)
    cuvit.rotary(x, at, turns, x, cuvit.rotary_problem(IMAGES, TOKENS, 1, 2, [1]))
    alone = torch.empty_like(one)
    cuvit.rotary(one, at, turns, alone, cuvit.rotary_problem(1, TOKENS, 1, 2, [1]))
    assert not torch.equal(alone, one) and images_are(x, alone)


def test_qk_norm_and_its_gradients():
    """52 GB. The long sums: a lane, which is a head of two, adds the 2^22 tokens
    of its workgroup in 2^14 rounds, each rounding what is summed; the rest as in
    the smaller cases."""
    g = support.seeded(2)
    qkv, grad = (support.normal(g, 1, TOKENS, 3, 2, dtype=torch.bfloat16) for _ in range(2))
    at, turns, gamma = positions_of(g, TOKENS, 1), ladder([1]), support.normal(g, 2, mean=1.0)
    many, single = (cuvit.qk_norm_problem(n, TOKENS, 1, 2, [1]) for n in (IMAGES, 1))
    there = [t.to(DEV) for t in (gamma, gamma, at, turns)]

    x, d = (t.to(DEV).repeat(IMAGES, 1, 1, 1) for t in (qkv, grad))
    sums = [torch.full((2,), 7.0, device=DEV) for _ in range(4)]
    workspace = torch.full((cuvit.qk_norm_rotary_workspace(many),), 255, dtype=torch.uint8, device=DEV)
    cuvit.qk_norm_rotary_backward(x, *there, d, d, many, workspace=workspace, grad_q_gamma=sums[0],
                                  grad_k_gamma=sums[1], grad_q_beta=sums[2], grad_k_beta=sums[3])
    alone = grad.to(DEV)
    cuvit.qk_norm_rotary_backward(qkv.to(DEV), *there, alone, alone, single)
    assert not torch.equal(alone.cpu(), grad) and images_are(d, alone)
    _, _, d_gamma, size_gamma, d_beta, size_beta = support.qk_norm_gradients(
        qkv, grad, 1, 1, False, 1.0e-6, [gamma, gamma], (at, turns, [1], False))
    unit = 2.0 ** -17 + (2 ** 14 + 305) * support.ARITHMETIC
    assert support.worst(torch.stack(sums[:2]), IMAGES * d_gamma, unit * IMAGES * size_gamma) <= 1.0
    assert support.worst(torch.stack(sums[2:]), IMAGES * d_beta, unit * IMAGES * size_beta) <= 1.0
    del d

    cuvit.qk_norm_rotary(x, *there, x, many)
    alone = torch.empty_like(qkv, device=DEV)
    cuvit.qk_norm_rotary(qkv.to(DEV), *there, alone, single)
    assert images_are(x, alone)


def test_strides_that_no_tensor_holds_are_refused():
    x = torch.full((2, 5, 3, 64), 7.0, device=DEV)
    out = torch.full_like(x, 7.0)
    at, turns = torch.zeros(5, 1, device=DEV), torch.zeros(32, device=DEV)
    for name in ("image", "token", "head"):
        for stride in (2 ** 40, 2 ** 62, 2 ** 63 - 1):
            problem = cuvit.rotary_problem(2, 5, 3, 64, [32])
            setattr(problem.input, name, stride)
            assert cuvit._native_calls.rotary(x, at, turns, out, problem, None, None) == -1
            with pytest.raises(cuvit.InvalidArgument, match="x holds 1920 elements"):
                cuvit.rotary(x, at, turns, out, problem)
    assert bool((out == 7.0).all())
