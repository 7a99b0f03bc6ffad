"""Attention over packed sequences and its gradients by every kernel that the rules can
choose (kernels/packed_choice.hpp): each division of the work at each width of heads, whole
widths and cut ones. test_packed_choice_cpu.py looks up which kernels these calls reach."""

from __future__ import annotations

import pytest
import torch

from packed_support import Packed
from test_packed_attention_gpu import TYPES, Call, both, check_forward, operands

pytestmark = pytest.mark.gpu

HEAD_DIMS = [24, 32, 64, 80, 96, 128, 200, 256]
CAUSAL = pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])

# (queries, keys, heads, kv_heads) of the forward's divisions; None: the queries' own.
# Sequences of several blocks of keys among short ones, groups of heads, tiles cut by the
# end of a sequence.
FORWARD = {
    "few": ([70, 9, 101], None, 4, 2),
    "middle": ([300, 150, 70, 1, 33], None, 24, 12),
    "middle_single_queries": ([1] * 22, [50, 1, 190] * 7 + [0], 12, 12),
    "large": ([290] + [20, 45, 64, 33, 70] * 7 + [0, 1], None, 24, 12),
    "parts": ([2, 1, 3], [3000, 40, 700], 4, 2),
}


@TYPES
@CAUSAL
@pytest.mark.parametrize("head_dim", HEAD_DIMS)
@pytest.mark.parametrize("division", FORWARD)
def test_forward(cuvit, device, dtype, causal, head_dim, division):
    queries, keys, heads, kv_heads = FORWARD[division]
    p = Packed(queries, heads, head_dim, kv_heads=kv_heads, keys=keys, causal=causal)
    q, k, v = operands(p, dtype, head_dim + 50)
    call = Call(cuvit, device, p, q, k, v)
    call.forward()
    check_forward(call, q, k, v)


# Of the gradients: {name: (queries, keys, heads, kv_heads)}.
GRADIENTS = {
    "alone": ([70, 9, 101], None, 4, 2),             # bf16: none share a tile
    "four": ([600, 530], None, 4, 2),                # all four wavefronts share one; pairs above 128
    "pairs_of_rows": ([64], [512], 256, 256),        # bf16: pairs
    "pairs_of_keys": ([512], [64], 256, 256),
}


@TYPES
@CAUSAL
@pytest.mark.parametrize("head_dim", HEAD_DIMS)
@pytest.mark.parametrize("division", ["alone", "four"])
def test_gradients(cuvit, device, dtype, causal, head_dim, division):
    queries, keys, heads, kv_heads = GRADIENTS[division]
    both(cuvit, device, Packed(queries, heads, head_dim, kv_heads=kv_heads, keys=keys, causal=causal), dtype,
         seed=head_dim)


@pytest.mark.parametrize("head_dim", [32, 56, 96, 128, 256])
@pytest.mark.parametrize("division", ["pairs_of_rows", "pairs_of_keys"])
def test_gradients_by_pairs(cuvit, device, head_dim, division):
    """Many heads; causal with fewer queries than keys, all keys with more."""
    queries, keys, heads, kv_heads = GRADIENTS[division]
    both(cuvit, device, Packed(queries, heads, head_dim, kv_heads=kv_heads, keys=keys, causal=division == "pairs_of_rows"),
         torch.bfloat16, seed=head_dim)
