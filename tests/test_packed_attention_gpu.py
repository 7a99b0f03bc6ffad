"""Attention over packed sequences and its gradients on the GPU against the 64-bit
formula (packed_support.py), at the lengths, layouts and values where they can go wrong."""

from __future__ import annotations

import math
import threading

import pytest
import torch

from blocks_support import normal, seeded, worst
from packed_support import Packed, forward, gradients

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def numbers(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


class Call:
    """One problem's operands on the GPU, results prefilled, and its two calls."""

    def __init__(self, cuvit, device, p, q, k, v, projection=False, sentinel=7.0):
        self.cuvit, self.p, self.projection = cuvit, p, projection
        dtype = q.dtype
        self.problem = cuvit.packed_attention_problem(len(p.queries), p.tokens, p.heads, p.head_dim,
                                                      kv_heads=p.kv_heads, kv_tokens=p.kv_tokens, causal=p.causal,
                                                      projection=projection)
        if p.scale != 1.0 / math.sqrt(p.head_dim):
            self.problem.scale = p.scale
        if projection:
            self.operands = [torch.cat([q, k, v], dim=1).to(device), None, None]
        else:
            self.operands = [x.to(device) for x in (q, k, v)]
        self.starts = numbers(p.starts, device)
        self.caches = {}
        if p.own_keys:
            self.caches["kv_starts"] = numbers(p.kv_starts, device)
        if p.rooms != p.keys:
            self.caches["kv_lengths"] = numbers(p.keys, device)
        self.out = torch.full((p.tokens, p.heads, p.head_dim), sentinel, dtype=dtype, device=device)
        self.lse = torch.full((p.tokens, p.heads), sentinel, device=device)
        self.grads = [None if x is None else torch.full_like(x, sentinel) for x in self.operands]
        self.workspace = self._bytes(cuvit.packed_attention_workspace(self.problem), device)
        self.backward_workspace = self._bytes(cuvit.packed_attention_backward_workspace(self.problem), device)

    @staticmethod
    def _bytes(count, device):
        return torch.full((count,), 255, dtype=torch.uint8, device=device) if count else None

    def forward(self, **options):
        self.cuvit.packed_attention(*self.operands, self.starts, self.out, self.problem, lse=self.lse,
                                    workspace=self.workspace, **self.caches, **options)

    def backward(self, grad, **options):
        self.cuvit.packed_attention_backward(*self.operands, self.starts, self.out, self.lse, grad, *self.grads,
                                             self.problem, workspace=self.backward_workspace, **self.caches, **options)

    def gradients(self):
        if not self.projection:
            return self.grads
        p = self.p
        return list(self.grads[0].split([p.heads, p.kv_heads, p.kv_heads], dim=1))


def operands(p, dtype, seed, scale=1.0):
    generator = seeded(seed)
    return (normal(generator, p.tokens, p.heads, p.head_dim, scale=scale, dtype=dtype),
            normal(generator, p.kv_tokens, p.kv_heads, p.head_dim, scale=scale, dtype=dtype),
            normal(generator, p.kv_tokens, p.kv_heads, p.head_dim, dtype=dtype))


def inside(p, count, keys=False):
    """Which rows belong to a sequence."""
    rows = torch.zeros(count, dtype=torch.bool)
    for queries, seen in p.sequences():
        rows[seen if keys else queries] = True
    return rows


def check_forward(call, q, k, v, sentinel=7.0):
    p = call.p
    expected, bound, lse, lse_bound = forward(p, q, k, v, q.dtype)
    rows = inside(p, p.tokens)
    out, produced_lse = call.out.cpu(), call.lse.cpu()
    assert worst(out[rows], expected[rows], bound[rows]) <= 1.0
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(produced_lse) & rows[:, None], empty & rows[:, None])
    some = rows[:, None] & ~empty
    assert worst(produced_lse[some], lse[some], lse_bound[some]) <= 1.0
    assert bool((out[~rows] == sentinel).all()) and bool((produced_lse[~rows] == sentinel).all())


def check_backward(call, q, k, v, grad, sentinel=7.0):
    p = call.p
    expected, bounds = gradients(p, q, k, v, grad, q.dtype)
    for i, produced in enumerate(call.gradients()):
        rows = inside(p, produced.shape[0], keys=i > 0)
        produced = produced.cpu()
        assert worst(produced[rows], expected[i][rows], bounds[i][rows]) <= 1.0, "qkv"[i]
        assert bool((produced[~rows] == sentinel).all()), "qkv"[i]


def both(cuvit, device, p, dtype, seed=1, projection=False, scale=1.0):
    q, k, v = operands(p, dtype, seed, scale)
    call = Call(cuvit, device, p, q, k, v, projection)
    call.forward()
    check_forward(call, q, k, v)
    grad = normal(seeded(seed + 1), p.tokens, p.heads, p.head_dim, dtype=dtype)
    call.backward(grad.to(device))
    check_backward(call, q, k, v, grad)
    return call


LENGTHS = [[197], [1], [0, 5, 0, 1, 33, 64, 65, 0], [300, 31, 128, 129], [2] * 70]


@TYPES
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=[str(x)[:16] for x in LENGTHS])
def test_lengths(cuvit, device, dtype, causal, lengths):
    both(cuvit, device, Packed(lengths, 3, 64, causal=causal), dtype, projection=True)


@TYPES
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("head_dim", [8, 32, 40, 64, 72, 80, 96, 104, 128, 136, 200, 256])
def test_widths(cuvit, device, dtype, causal, head_dim):
    both(cuvit, device, Packed([70, 9, 101], 4, head_dim, kv_heads=2, causal=causal), dtype, seed=head_dim)


@TYPES
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (2, 1), (6, 2), (12, 4), (16, 1), (5, 5), (7, 1)])
def test_shared_heads(cuvit, device, dtype, causal, heads, kv_heads):
    both(cuvit, device, Packed([50, 3, 77], heads, 64, kv_heads=kv_heads, causal=causal), dtype, projection=True)


OTHER_KEYS = [([1, 1, 1], [5, 0, 170]), ([1, 2, 1], [1, 300, 2]), ([3, 40, 2, 0], [1, 40, 700, 20]),
              ([200, 5], [0, 130]), ([1], [1200]), ([64, 64], [64, 65])]


@TYPES
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("queries,keys", OTHER_KEYS, ids=[str(x)[:24] for x in OTHER_KEYS])
def test_keys_of_their_own(cuvit, device, dtype, causal, queries, keys):
    """Fewer and more queries than keys (causal: the first ones then see none), no
    keys, no queries: zeros and -infinity, and zero gradients of unseen keys."""
    both(cuvit, device, Packed(queries, 6, 64, kv_heads=2, keys=keys, causal=causal), dtype)


@TYPES
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(12, 4, 128), (8, 8, 64), (16, 1, 80), (3, 3, 256)])
@pytest.mark.parametrize("queries", [1, 3])
def test_caches_with_room(cuvit, device, dtype, heads, kv_heads, head_dim, queries):
    """What lies in a cache behind the filled keys is never seen, NaN included."""
    keys = [queries, 40, 1000, 129, 64]
    p = Packed([queries] * 5, heads, head_dim, kv_heads=kv_heads, keys=keys, rooms=[1024] * 5, causal=True)
    q, k, v = operands(p, dtype, 3)
    outside = ~inside(p, p.kv_tokens, keys=True)
    k[outside], v[outside] = math.nan, math.inf
    call = Call(cuvit, device, p, q, k, v)
    call.forward()
    k[outside], v[outside] = 0.0, 0.0
    check_forward(call, q, k, v)
    grad = normal(seeded(4), p.tokens, heads, head_dim, dtype=dtype)
    call.backward(grad.to(device))
    check_backward(call, q, k, v, grad)


@TYPES
@pytest.mark.parametrize("queries,keys,heads,kv_heads,head_dim", [
    ([1] * 16, [2000] * 15 + [700], 12, 4, 128),   # parts of the keys, joined
    ([2] * 3, [5000, 0, 130], 4, 2, 64),
    ([1], [6000], 2, 1, 80),
    ([1] * 90, [60] * 90, 12, 12, 64),             # many single queries: pairs of wavefronts
    ([150] * 40, [150] * 40, 12, 4, 64),           # whole tiles
], ids=["parts", "parts_of_uneven_keys", "parts_of_one", "pairs", "tiles"])
def test_divisions(cuvit, device, dtype, queries, keys, heads, kv_heads, head_dim):
    both(cuvit, device, Packed(queries, heads, head_dim, kv_heads=kv_heads, keys=keys, causal=True), dtype)


@TYPES
def test_bad_values_in_parts_of_the_keys(cuvit, device, dtype):
    """As below, where a query's keys are in parts: rows that meet them are taken again."""
    p = Packed([3], 2, 64, keys=[4000], causal=True)
    q, k, v = operands(p, dtype, 22)
    clean, bound, lse, lse_bound = forward(p, q, k, v, dtype)
    v[3999], k[3998, 0] = math.inf, math.nan
    call = Call(cuvit, device, p, q, k, v)
    assert cuvit.packed_attention_workspace(call.problem) > 0
    call.forward()
    out = call.out.cpu()
    assert worst(out[0], clean[0], bound[0]) <= 1.0
    assert worst(call.lse.cpu()[0], lse[0], lse_bound[0]) <= 1.0
    assert bool(torch.isnan(out[1, 0]).all()) and worst(out[1, 1], clean[1, 1], bound[1, 1]) <= 1.0
    assert not bool(torch.isfinite(out[2]).any())


@TYPES
def test_no_keys_and_no_queries_at_all(cuvit, device, dtype):
    """kv_tokens 0: zeros, -infinity and zero gradients; tokens 0: zero gradients of the keys."""
    starts = numbers([0, 2, 5], device)
    nothing = numbers([0, 0, 0], device)
    p = cuvit.packed_attention_problem(2, 5, 4, 64, kv_heads=2, kv_tokens=0)
    x = torch.ones(5, 4, 64, dtype=dtype, device=device)
    out, lse = torch.full_like(x, 7.0), torch.full((5, 4), 7.0, device=device)
    cuvit.packed_attention(x, None, None, starts, out, p, kv_starts=nothing, lse=lse)
    assert bool((out == 0.0).all()) and bool((lse == -math.inf).all())
    grad = torch.full_like(x, 7.0)
    size = cuvit.packed_attention_backward_workspace(p)
    cuvit.packed_attention_backward(x, None, None, starts, out, lse, x, grad, None, None, p, kv_starts=nothing,
                                    workspace=torch.zeros(size, dtype=torch.uint8, device=device))
    assert bool((grad == 0.0).all())
    p = cuvit.packed_attention_problem(2, 0, 4, 64, kv_heads=2, kv_tokens=5)
    k = torch.ones(5, 2, 64, dtype=dtype, device=device)
    grads = [torch.full_like(k, 7.0) for _ in range(2)]
    assert cuvit.packed_attention_backward_workspace(p) == 0
    cuvit.packed_attention(None, k, k, nothing, None, p, kv_starts=starts, bf16=dtype == torch.bfloat16)
    cuvit.packed_attention_backward(None, k, k, nothing, None, None, None, None, *grads, p, kv_starts=starts,
                                    bf16=dtype == torch.bfloat16)
    assert all(bool((g == 0.0).all()) for g in grads)


@TYPES
def test_rows_outside_are_not_read(cuvit, device, dtype):
    """NaN behind the last sequence and in other sequences stays there."""
    p = Packed([65, 30, 100], 2, 64, causal=True, spare=40)
    q, k, v = operands(p, dtype, 6)
    grad = normal(seeded(7), *q.shape, dtype=dtype)
    bad = [x.clone() for x in (q, k, v)]
    for x in bad:
        x[p.starts[-1]:] = math.nan
        x[p.starts[1]:p.starts[2]] = math.nan
    call = Call(cuvit, device, p, *bad)
    call.forward()
    call.backward(grad.to(device))
    out = call.out.cpu()
    assert bool(torch.isnan(out[p.starts[1]:p.starts[2]]).all())
    keep = torch.cat([torch.arange(0, 65), torch.arange(95, 195)])
    expected, bound, _, _ = forward(p, q, k, v, dtype)
    assert worst(out[keep], expected[keep], bound[keep]) <= 1.0
    expected, bounds = gradients(p, q, k, v, grad, dtype)
    for x, e, b in zip(call.gradients(), expected, bounds):
        assert worst(x.cpu()[keep], e[keep], b[keep]) <= 1.0


@TYPES
def test_bad_values_of_later_keys(cuvit, device, dtype):
    """Causal: a query's result does not know keys behind it, whatever they hold."""
    p = Packed([40, 130], 2, 80, causal=True)
    q, k, v = operands(p, dtype, 8)
    clean, bound, lse, lse_bound = forward(p, q, k, v, dtype)
    k[20], v[21] = math.nan, math.inf
    v[40 + 70], k[40 + 100] = math.nan, math.inf
    call = Call(cuvit, device, p, q, k, v)
    call.forward()
    out, produced = call.out.cpu(), call.lse.cpu()
    keep = torch.cat([torch.arange(0, 20), torch.arange(40, 110)])
    assert worst(out[keep], clean[keep], bound[keep]) <= 1.0
    assert worst(produced[keep], lse[keep], lse_bound[keep]) <= 1.0
    assert bool(torch.isnan(out[20:40]).all()) and bool(torch.isnan(out[110:140]).all())


@TYPES
@pytest.mark.parametrize("scale", [30.0, 1e-3], ids=["large_logits", "small_logits"])
def test_logits(cuvit, device, dtype, scale):
    """Logits of thousands leave one weight of about 1; of a millionth, equal ones."""
    p = Packed([100, 65], 3, 64)
    q, k, v = operands(p, dtype, 9, scale)
    call = Call(cuvit, device, p, q, k, v)
    call.forward()
    check_forward(call, q, k, v)


@TYPES
def test_a_scale(cuvit, device, dtype):
    both(cuvit, device, Packed([90, 17], 2, 72, scale=0.5), dtype)


@TYPES
def test_largest_values(cuvit, device, dtype):
    """Sums of weights times values beyond the type's largest are not infinite."""
    p = Packed([80, 33], 2, 64)
    q, k, v = operands(p, dtype, 10)
    v = (v.float().clamp(-1.0, 1.0) * 3.0e38).to(dtype)
    call = Call(cuvit, device, p, q, k, v)
    call.forward()
    check_forward(call, q, k, v)


@TYPES
def test_no_logit_above_minus_infinity(cuvit, device, dtype):
    p = Packed([10, 50], 1, 64)
    q, k, v = operands(p, dtype, 11)
    q = q.abs()
    k[:10] = -math.inf
    k[30:] = -math.inf  # of the second sequence's keys some stay
    call = Call(cuvit, device, p, q, k, v)
    call.forward()
    out, lse = call.out.cpu(), call.lse.cpu()
    assert bool(torch.isnan(out[:10]).all())
    assert bool((lse[:10] == -math.inf).all())
    rest = Packed([20], 1, 64, spare=0)
    both_k, both_v = k[10:30], v[10:30]
    for row in (10, 59):
        x = (q[row, 0].double() @ both_k[:, 0].double().t()) / 8.0
        y = torch.softmax(x, 0) @ both_v[:, 0].double()
        _, bound, _, _ = forward(rest, q[row:row + 1].expand(20, -1, -1), both_k, both_v, dtype)
        assert worst(out[row, 0], y, bound[0, 0]) <= 1.0


@TYPES
def test_strides(cuvit, device, dtype):
    """Heads first, wide rows, and results between others' values."""
    p = Packed([70, 45], 4, 64, kv_heads=2, causal=True)
    q, k, v = operands(p, dtype, 12)
    grad = normal(seeded(13), *q.shape, dtype=dtype)
    plain = Call(cuvit, device, p, q, k, v)
    plain.forward()
    plain.backward(grad.to(device))
    call = Call(cuvit, device, p, q, k, v)
    tokens = p.tokens
    pr = call.problem
    pr.q.token, pr.q.head = 64, 64 * tokens
    pr.k.token, pr.k.head = 320, 72
    pr.v.token, pr.v.head = 64, 64 * tokens + 16
    pr.out.token, pr.out.head = 600, 80

    def spread(x, strides, size):
        flat = torch.full((size,), 7.0, dtype=dtype, device=device)
        view = flat.as_strided(x.shape, (strides.token, strides.head, 1))
        view.copy_(x)
        return flat, view

    flats = [spread(x, s, 600 * tokens) for x, s in ((q, pr.q), (k, pr.k), (v, pr.v))]
    call.operands = [f for f, _ in flats]
    call.out, out_view = spread(torch.full_like(q, 7.0), pr.out, 600 * tokens)
    call.forward()
    assert torch.equal(out_view, plain.out) and torch.equal(call.lse, plain.lse)
    grad_flat, _ = spread(grad, pr.out, 600 * tokens)
    results = [spread(torch.full_like(x, 7.0), s, 600 * tokens) for x, s in ((q, pr.q), (k, pr.k), (v, pr.v))]
    call.grads = [f for f, _ in results]
    call.backward(grad_flat)
    for (flat, view), expected, x in zip(results, plain.grads, (q, k, v)):
        assert torch.equal(view, expected)
        assert int((flat != 7.0).sum()) <= x.numel()
    assert int((call.out != 7.0).sum()) <= q.numel()


@TYPES
@pytest.mark.parametrize("starts", [[5, 3, 40, 10, 60], [-9, 20, 20, 1000, 60], [70, 80, 90, 100, 110],
                                    [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0, 9]])
def test_starts_that_do_not_fit(cuvit, device, dtype, starts):
    """Cut to the operands: nothing outside them is read or written."""
    p = Packed([20, 20, 10, 14], 2, 64, spare=0)
    q, k, v = operands(p, dtype, 14)
    call = Call(cuvit, device, p, q, k, v)
    guard = torch.full((3, 4096, 2, 64), 7.0, dtype=dtype, device=device)
    call.out = guard[1, :64]
    call.starts.copy_(numbers(starts, device))
    call.caches["kv_lengths"] = numbers([2 ** 31 - 1, -5, 3, 2 ** 31 - 1], device)
    call.forward()
    call.backward(torch.ones_like(call.out))
    torch.cuda.synchronize()
    assert bool((guard[0] == 7.0).all()) and bool((guard[2] == 7.0).all()) and bool((guard[1, 64:] == 7.0).all())


@TYPES
def test_same_bits_again(cuvit, device, dtype):
    p = Packed([300, 70, 1, 129], 6, 64, kv_heads=2, causal=True)
    q, k, v = operands(p, dtype, 15)
    grad = normal(seeded(16), *q.shape, dtype=dtype).to(device)
    results = []
    for _ in range(3):
        call = Call(cuvit, device, p, q, k, v)
        call.forward()
        call.backward(grad)
        results.append([call.out, call.lse] + call.grads)
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@TYPES
def test_a_sequence_alone_and_among_others(cuvit, device, dtype):
    """Equal bits wherever a sequence lies, in a batch of one or of many."""
    p = Packed([77, 200, 50], 3, 64)
    q, k, v = operands(p, dtype, 17)
    whole = Call(cuvit, device, p, q, k, v)
    whole.forward()
    rows = slice(77, 277)
    one = Packed([200], 3, 64, spare=0)
    alone = Call(cuvit, device, one, q[rows], k[rows], v[rows])
    alone.forward()
    assert torch.equal(alone.out, whole.out[rows]) and torch.equal(alone.lse, whole.lse[rows])


@TYPES
def test_streams_threads_and_graphs(cuvit, device, dtype):
    p = Packed([100, 31, 64], 4, 64, kv_heads=2, causal=True)
    q, k, v = operands(p, dtype, 18)
    grad = normal(seeded(19), *q.shape, dtype=dtype).to(device)
    expected = Call(cuvit, device, p, q, k, v)
    expected.forward()
    expected.backward(grad)
    torch.cuda.synchronize()

    def same(call):
        torch.cuda.synchronize()
        return (torch.equal(call.out, expected.out) and torch.equal(call.lse, expected.lse)
                and all(torch.equal(a, b) for a, b in zip(call.grads, expected.grads)))

    # Another stream, as an argument and as the current one.
    stream = torch.cuda.Stream()
    call = Call(cuvit, device, p, q, k, v)
    torch.cuda.synchronize()
    call.forward(stream=stream)
    with torch.cuda.stream(stream):
        call.backward(grad)
    assert same(call)

    # Several threads, a workspace each.
    calls = [Call(cuvit, device, p, q, k, v) for _ in range(4)]
    torch.cuda.synchronize()

    def work(c):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                c.forward()
                c.backward(grad)

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(same(c) for c in calls)

    # Captured, replayed with other lengths and values in the same memory, and back.
    call = Call(cuvit, device, p, q, k, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call.forward()
        call.backward(grad)
    other = Packed([3, 150, 42], 4, 64, kv_heads=2, causal=True)
    others = operands(other, dtype, 20)
    moved = Call(cuvit, device, other, *others)
    moved.forward()
    moved.backward(grad)
    for turn in range(4):
        use, values = (p, (q, k, v)) if turn % 2 == 0 else (other, others)
        for x, y in zip(call.operands, values):
            x.copy_(y)
        call.starts.copy_(numbers(use.starts, device))
        for x in [call.out, call.lse] + call.grads:
            x.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        wanted = expected if turn % 2 == 0 else moved
        assert torch.equal(call.out, wanted.out) and torch.equal(call.lse, wanted.lse)
        assert all(torch.equal(a, b) for a, b in zip(call.grads, wanted.grads))


def test_offsets_beyond_32_bits(cuvit, device):
    """A cache of 4.3 GB of keys: the first sequence's alone end 4.2 GB in."""
    room = 4_200_000
    p = Packed([1, 2], 2, 128, kv_heads=2, keys=[room, 300], causal=True, spare=0, rooms=[room, 300])
    k = torch.zeros(p.kv_tokens, 4, 128, dtype=torch.bfloat16, device=device)
    v = torch.zeros_like(k)
    generator = seeded(21)
    tail = 500  # random keys at the end of the first sequence, all of the second's
    for x in (k, v):
        x[room - tail:] = normal(generator, tail + 300, 4, 128, dtype=torch.bfloat16).to(device)
    q = normal(generator, 3, 2, 128, dtype=torch.bfloat16)
    problem = cuvit.packed_attention_problem(2, 3, 2, 128, kv_heads=2, kv_tokens=p.kv_tokens, causal=True)
    problem.k.token = problem.v.token = 512
    out = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=device)
    lse = torch.zeros(3, 2, device=device)
    size = cuvit.packed_attention_workspace(problem)
    cuvit.packed_attention(q.to(device), k, v, numbers([0, 1, 3], device), out, problem,
                           kv_starts=numbers(p.kv_starts, device), lse=lse,
                           workspace=torch.zeros(size, dtype=torch.uint8, device=device) if size else None)
    small = Packed([2], 2, 128, keys=[300], causal=True, spare=0)
    second = [x[room:, :2].cpu() for x in (k, v)]
    expected, bound, _, _ = forward(small, q[1:], *second, torch.bfloat16)
    assert worst(out[1:].cpu(), expected, bound) <= 1.0
    # The first: keys of zeros have logits of 0 and values of 0.
    first = [x[room - tail:room, :2].cpu().double() for x in (k, v)]
    for h in range(2):
        x = q[0, h].double() @ first[0][:, h].t() / math.sqrt(128)
        total = torch.exp(x).sum() + (room - tail)
        assert abs(float(lse[0, h]) - float(torch.log(total))) < 1e-4  # 4.2 M terms of 1 in fp32 lanes' sums
        y = torch.exp(x) @ first[1][:, h] / total
        assert float((out[0, h].cpu().double() - y).abs().max()) <= 2.0 ** -7 * float((torch.exp(x) @ first[1][:, h].abs()).max() / total)
