"""Attention over packed sequences where rows, values and sizes are at an edge."""

from __future__ import annotations

import math

import pytest
import torch

from packed_support import Packed, forward
from blocks_support import worst
from test_packed_attention_gpu import TYPES, Call, operands

pytestmark = pytest.mark.gpu


# Causal calls with sequences of more queries than keys, by each division of the work.
NO_KEYS = [
    ("few", [40], [10], 2, 2, 64),
    ("pairs", [3] * 90, [2] * 90, 12, 12, 64),
    ("tiles", [150] * 40, [60] * 40, 12, 4, 64),
    ("parts", [3, 3], [6000, 2], 2, 1, 64),
]


@TYPES
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan], ids=["inf", "-inf", "nan"])
@pytest.mark.parametrize("queries,keys,heads,kv_heads,head_dim", [c[1:] for c in NO_KEYS], ids=[c[0] for c in NO_KEYS])
def test_rows_without_keys_beside_bad_values(cuvit, device, dtype, bad, queries, keys, heads, kv_heads, head_dim):
    """Zeros and -infinity, whatever the values hold that other rows of the tile see; rows
    that see keys, but none of the bad ones, are as they were."""
    p = Packed(queries, heads, head_dim, kv_heads=kv_heads, keys=keys, causal=True)
    q, k, v = operands(p, dtype, 31)
    clean, bound, lse, lse_bound = forward(p, q, k, v, dtype)
    unseen = torch.zeros(p.tokens, dtype=torch.bool)
    untouched = torch.zeros(p.tokens, dtype=torch.bool)
    for rows, seen in p.sequences():
        count, n = rows.stop - rows.start, seen.stop - seen.start
        at = n // 2  # the bad key
        v[seen.start + at] = bad
        last = torch.arange(count) + n - count  # the last key that a query sees
        unseen[rows] = last < 0
        untouched[rows] = (last >= 0) & (last < at)
    assert bool(unseen.any())
    call = Call(cuvit, device, p, q, k, v)
    call.forward()
    out, produced = call.out.cpu(), call.lse.cpu()
    assert bool((out[unseen] == 0.0).all())
    assert bool((produced[unseen] == -math.inf).all())
    assert worst(out[untouched], clean[untouched], bound[untouched]) <= 1.0
    assert worst(produced[untouched], lse[untouched], lse_bound[untouched]) <= 1.0
