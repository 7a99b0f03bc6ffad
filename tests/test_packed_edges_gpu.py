"""Attention over packed sequences where rows, values and sizes are at an edge."""

from __future__ import annotations

import math

import pytest
import torch

from packed_support import Packed, forward
from blocks_support import seeded, worst
from test_packed_attention_gpu import TYPES, Call, check_forward, operands

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


@pytest.mark.parametrize("queries", [1, 33])
def test_the_longest_cache(cuvit, device, queries):
    """2^31 - 4096 keys of 8 values in bf16, 34 GB, in parts that are joined. Keys and
    values are zeros but for the last key's, whose logit is 30: only the last query sees
    it, and 2^31 weights of exp(-30), 2e-4 in all, beside it; the others sum ones."""
    keys = 2 ** 31 - 4096
    if torch.cuda.mem_get_info()[0] < 80e9:
        pytest.skip("needs 80 GB of memory")
    k = torch.zeros(keys, 1, 8, dtype=torch.bfloat16, device=device)
    v = torch.zeros_like(k)
    k[-1], v[-1] = 4.0, torch.arange(1, 9, device=device).to(torch.bfloat16)
    q = torch.ones(queries, 1, 8, dtype=torch.bfloat16, device=device)
    p = cuvit.packed_attention_problem(1, queries, 1, 8, kv_tokens=keys, scale=30.0 / 32.0, causal=True)
    out = torch.full_like(q, 7.0)
    lse = torch.full((queries, 1), 7.0, device=device)
    size = cuvit.packed_attention_workspace(p)
    assert size > 0
    cuvit.packed_attention(q, k, v, torch.tensor([0, queries], dtype=torch.int32, device=device), out, p,
                           kv_starts=torch.tensor([0, keys], dtype=torch.int32, device=device), lse=lse,
                           workspace=torch.zeros(size, dtype=torch.uint8, device=device))
    out, lse = out[:, 0].cpu().double(), lse[:, 0].cpu().double()
    del k, v
    torch.cuda.empty_cache()
    # A lane's sums are multiples of 16 below 2^28, or of 1 below 2^24: exact. A weight of
    # exp(-30) is off by its argument's rounding, 2^-24 of 43 a factor of it and as many
    # again in the maxima, below 2^-14 in all; the log-sum-exp by its factors' roundings.
    small = (keys - 1) * math.exp(-30.0)
    value = torch.arange(1, 9).double() / (1.0 + small)
    assert worst(out[-1], value, (2.0 ** -8 + 2.0 ** -14) * value) <= 1.0
    assert abs(float(lse[-1]) - (30.0 + math.log1p(small))) <= 2.0 ** -14 * small + 8 * 2.0 ** -24 * 30.0
    if queries > 1:
        seen = keys - queries + torch.arange(1, queries).double()
        assert bool((out[:-1] == 0.0).all())
        assert float((lse[:-1] - torch.log(seen)).abs().max()) <= 8 * 2.0 ** -24 * 30.0


@TYPES
@pytest.mark.parametrize("scale", [2.0 ** 127, 2.0 ** -126])
def test_scales_at_their_limits(cuvit, device, dtype, scale):
    """At the largest, products of 2^-126 times 0 to 4, exact ones, give logits of 0 to 8;
    at the smallest the logits vanish and every key weighs the same."""
    p = Packed([40, 70], 2, 64, scale=scale, causal=True)
    q, k, v = operands(p, dtype, 33)
    if scale > 1.0:
        multiples = torch.randint(0, 5, k.shape[:2], generator=seeded(34)).to(dtype)
        q.zero_()[..., 0] = 2.0 ** -100
        k.zero_()[..., 0] = multiples * 2.0 ** -26
    call = Call(cuvit, device, p, q, k, v)
    call.forward()
    check_forward(call, q, k, v)


class Guarded:
    """A tensor of `shape` between two stretches of memory that nobody may write."""

    def __init__(self, shape, dtype, device, value, margin=1 << 18):
        size = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
        self.memory = torch.full((2 * margin + size,), 0x5A, dtype=torch.uint8, device=device)
        self.tensor = self.memory[margin:margin + size].view(dtype).view(shape)
        self.tensor.fill_(value)
        self.margin = margin

    def untouched(self):
        sides = torch.cat([self.memory[:self.margin], self.memory[-self.margin:]])
        return bool((sides == 0x5A).all())


GUARDED = [  # queries, keys, heads, kv_heads, head_dim: each division of the forward and the gradients
    ([20, 20, 10, 14], None, 2, 2, 64),
    ([70, 9, 101], None, 4, 2, 128),
    ([2, 1, 3], [3000, 40, 700], 4, 2, 80),
    ([300, 150, 70, 1, 33], None, 24, 12, 64),
    ([290] + [20, 45, 64, 33, 70] * 7 + [0, 1], None, 24, 12, 32),
    ([600, 530], None, 4, 2, 96),
    ([64], [512], 256, 256, 32),
    ([512], [64], 256, 256, 32),
]


@TYPES
@pytest.mark.parametrize("fits", [True, False], ids=["starts", "starts_that_do_not_fit"])
@pytest.mark.parametrize("queries,keys,heads,kv_heads,head_dim", GUARDED, ids=[str(g[0])[:20] for g in GUARDED])
def test_nothing_beside_the_results_is_written(cuvit, device, dtype, fits, queries, keys, heads, kv_heads, head_dim):
    """out, lse, the three gradients and both workspaces, with sequences that the operands
    hold, and with starts and lengths that lead far outside them."""
    p = Packed(queries, heads, head_dim, kv_heads=kv_heads, keys=keys, causal=True, spare=0)
    q, k, v = operands(p, dtype, 35)
    call = Call(cuvit, device, p, q, k, v)
    out = Guarded(call.out.shape, dtype, device, 0.0)
    lse = Guarded(call.lse.shape, torch.float32, device, 0.0)
    grads = [Guarded(x.shape, dtype, device, 0.0) for x in call.operands]
    sizes = [cuvit.packed_attention_workspace(call.problem), cuvit.packed_attention_backward_workspace(call.problem)]
    workspaces = [Guarded((size,), torch.uint8, device, 255) if size else None for size in sizes]
    call.out, call.lse, call.grads = out.tensor, lse.tensor, [g.tensor for g in grads]
    call.workspace, call.backward_workspace = (w.tensor if w is not None else None for w in workspaces)
    if not fits:
        count = len(queries)
        call.starts.copy_(torch.tensor(([-9, 2 ** 31 - 1, p.tokens - 3, p.tokens + 100, -2 ** 31] * count)[:count + 1]))
        call.caches["kv_starts"] = torch.tensor(([5, p.kv_tokens + 64, -7, 2 ** 31 - 1] * count)[:count + 1],
                                                dtype=torch.int32, device=device)
        call.caches["kv_lengths"] = torch.tensor(([2 ** 31 - 1, 40, -5] * count)[:count], dtype=torch.int32, device=device)
    call.forward()
    call.backward(torch.ones_like(call.out))
    torch.cuda.synchronize()
    for name, guarded in (("out", out), ("lse", lse), ("grad_q", grads[0]), ("grad_k", grads[1]), ("grad_v", grads[2]),
                          ("workspace", workspaces[0]), ("backward workspace", workspaces[1])):
        assert guarded is None or guarded.untouched(), name


@TYPES
def test_a_captured_call_while_caches_fill(cuvit, device, dtype):
    """Single queries over caches with room, in parts: one graph replayed as the caches grow
    from nothing to full, with eager calls between the replays."""
    room, sequences, heads, kv_heads, head_dim = 3000, 3, 4, 2, 64
    full = Packed([1] * sequences, heads, head_dim, kv_heads=kv_heads, keys=[room - 1] * sequences,
                  rooms=[room] * sequences, causal=True, spare=0)
    q, k, v = operands(full, dtype, 41)
    call = Call(cuvit, device, full, q, k, v)
    assert cuvit.packed_attention_workspace(call.problem) > 0
    call.forward()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call.forward()
    for lengths in ([0, 0, 0], [1, 0, 2], [64, 65, 1], [127, 2999, 0], [500, 1280, 2048], [room, room, room]):
        p = Packed([1] * sequences, heads, head_dim, kv_heads=kv_heads, keys=lengths, rooms=[room] * sequences,
                   causal=True, spare=0)
        fresh = operands(p, dtype, 42 + sum(lengths))[0]
        eager = Call(cuvit, device, p, fresh, k, v)
        eager.caches["kv_lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
        eager.forward()
        call.operands[0].copy_(fresh)
        call.caches["kv_lengths"].copy_(eager.caches["kv_lengths"])
        call.out.fill_(7.0)
        call.lse.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(call.out, eager.out) and torch.equal(call.lse, eager.lse)
        call.p = p
        check_forward(call, fresh, k, v)
