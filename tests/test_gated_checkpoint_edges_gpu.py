"""Gated products that keep 8-bit codes, and the gradient from them, where sizes and memory
are at an edge."""

from __future__ import annotations

import pytest
import torch

from blocks_support import gated, normal, seeded, worst
from test_gated_checkpoint_gpu import TYPES, check_codes, kept
from test_packed_edges_gpu import Guarded

pytestmark = pytest.mark.gpu


@TYPES
@pytest.mark.parametrize("m,n", [(1, 1), (3, 17), (40, 96), (70, 40), (300, 129), (788, 1365), (3152, 2048)])
@pytest.mark.parametrize("with_bias", [True, False], ids=["bias", "none"])
def test_sums_of_nothing(cuvit, device, dtype, m, n, with_bias):
    """k 0: preactivations are the bias, or zeros."""
    generator = seeded(m + n)
    bias = normal(generator, 2 * n) if with_bias else None
    p = cuvit.gated_problem(m, n, 0)
    out = torch.full((m, n), 7.0, dtype=dtype, device=device)
    codes, scales = kept(p, cuvit, device)
    a, w = (torch.full((8,), 7.0, dtype=dtype, device=device) for _ in range(2))
    cuvit.gated_checkpoint_gemm(a, w, bias.to(device) if with_bias else None, out, codes, scales, p)
    nothing = [torch.zeros(rows, 1, dtype=dtype, device=device) for rows in (m, 2 * n)]
    expected, bound, z, _ = (x.cpu() for x in gated(*nothing, bias.to(device) if with_bias else None, 0, dtype))
    assert worst(out, expected, bound) <= 1.0
    check_codes(codes, scales, z, torch.zeros_like(z), n)


@TYPES
@pytest.mark.parametrize("m,n,k", [(1, 1, 8), (5, 33, 8), (66, 70, 37), (197, 683, 64), (788, 1365, 8), (3152, 2048, 8),
                                   (4616, 1000, 64)])
def test_nothing_beside_the_results_is_written(cuvit, device, dtype, m, n, k):
    generator = seeded(n)
    a, w = (normal(generator, rows, k, dtype=dtype).to(device) for rows in (m, 2 * n))
    p = cuvit.gated_problem(m, n, k)
    out = Guarded((m, n), dtype, device, 0.0)
    codes = Guarded((m, 2 * n), torch.uint8, device, 0)
    scales = Guarded((cuvit.gated_checkpoint_scales(p),), torch.uint8, device, 0)
    grad_pre, hidden = Guarded((m, 2 * n), dtype, device, 0.0), Guarded((m, n), dtype, device, 0.0)
    kept_codes = codes.tensor.view(torch.float8_e4m3fn), scales.tensor.view(torch.float8_e8m0fnu)
    cuvit.gated_checkpoint_gemm(a, w, None, out.tensor, *kept_codes, p)
    cuvit.gated_checkpoint_backward(*kept_codes, out.tensor, grad_pre.tensor, p, hidden=hidden.tensor)
    torch.cuda.synchronize()
    for name, guarded in (("out", out), ("codes", codes), ("scales", scales), ("grad", grad_pre), ("hidden", hidden)):
        assert guarded.untouched(), name
