"""A gated product of the largest k (13 GB of operands), and the gradient, which
has none."""

from __future__ import annotations

import pytest
import torch

import cuvit_amd as cuvit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_the_largest_depth():
    """Products at both ends and the middle of k, so sums are exact; NaN behind the
    operands stays out of them."""
    k = 2 ** 31 - 4096
    a = torch.zeros(k + 64, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(2 * k + 64, dtype=torch.bfloat16, device=DEV)
    a[k:], w[2 * k:] = float("nan"), float("nan")
    for place, left in ((0, 1.0), (k // 2 + 1, 2.0), (k - 1, 4.0)):
        a[place], w[place], w[k + place] = left, 1.0, -0.5
    out = torch.full((8,), 7.0, dtype=torch.bfloat16, device=DEV)
    pre = torch.full((8,), 7.0, dtype=torch.bfloat16, device=DEV)
    cuvit.gated_gemm(a[:k], w[:2 * k], None, out[:1], cuvit.gated_problem(1, 1, k, cuvit.GATE_GELU_TANH),
                     preactivations=pre[:2])
    assert pre.tolist() == [7.0, -3.5] + [7.0] * 6
    assert out.tolist() == [-24.5] + [7.0] * 7  # a gate of 7 passes whole


def test_the_gradient_does_not_use_k():
    z, d = torch.ones(2, 6, device=DEV), torch.ones(2, 3, device=DEV)
    results = [torch.empty_like(z) for _ in range(2)]
    for out, k in zip(results, (1, 2 ** 31 - 1)):
        cuvit.gated_backward(z, d, out, cuvit.gated_problem(2, 3, k))
    assert torch.equal(*results)
