"""Attention over packed sequences written out in 64 bits, and how far a kernel may
be from it.

The bounds count roundings: u = eps / 2 of the type, 2^-24 for fp32 arithmetic.
"""

from __future__ import annotations

import math

import torch

from blocks_support import ARITHMETIC, ROUNDING

EXPONENTIAL = 2.0 ** -21  # of exp2, its rounded argument's remainder and the rescaling products


class Packed:
    """Sequences of given lengths in operands with `spare` rows behind the last one."""

    def __init__(self, queries, heads, head_dim, kv_heads=None, keys=None, causal=False, spare=3, rooms=None,
                 scale=None):
        self.queries, self.heads, self.head_dim = list(queries), heads, head_dim
        self.kv_heads = kv_heads or heads
        self.own_keys = keys is not None
        self.keys = list(keys) if keys is not None else self.queries
        self.rooms = list(rooms) if rooms is not None else self.keys  # of each sequence's cache
        self.causal, self.spare = causal, spare
        self.scale = scale if scale is not None else 1.0 / math.sqrt(head_dim)
        self.starts = self._starts(self.queries)
        self.kv_starts = self._starts(self.rooms)
        self.tokens = self.starts[-1] + spare
        self.kv_tokens = self.kv_starts[-1] + spare

    @staticmethod
    def _starts(lengths):
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        return starts

    def sequences(self):
        for s, (n, keys) in enumerate(zip(self.queries, self.keys)):
            yield slice(self.starts[s], self.starts[s] + n), slice(self.kv_starts[s], self.kv_starts[s] + keys)

    def seen(self, n, keys):
        """[n, keys]: which keys a query sees."""
        if not self.causal:
            return torch.ones(n, keys, dtype=torch.bool)
        return torch.arange(keys)[None] <= torch.arange(n)[:, None] + (keys - n)

    def shared(self, head):
        return head * self.kv_heads // self.heads


def _weights(p, q, k):
    """Weights and log-sum-exps of one sequence and head, rows without keys 0 and
    -inf, and the relative error of a row's weights."""
    x = q @ k.t() * p.scale
    seen = p.seen(*x.shape)
    x = x.masked_fill(~seen, -math.inf)
    some = seen.any(dim=1) if x.shape[1] else torch.zeros(x.shape[0], dtype=torch.bool)
    lse = torch.logsumexp(x, dim=1) if x.shape[1] else torch.full((x.shape[0],), -math.inf, dtype=torch.float64)
    w = torch.where(seen & some[:, None], torch.exp(x - torch.where(some, lse, 0.0)[:, None]), 0.0)
    # A sum of head_dim products rounds as often; the scale, the exponent's argument and
    # the shift by the maximum once each, of numbers up to the largest logit's size.
    size = (q.abs() @ k.abs().t() * p.scale).masked_fill(~seen, 0.0)
    top = size.amax(dim=1) if size.shape[1] else torch.zeros(size.shape[0], dtype=torch.float64)
    return w, lse, (p.head_dim + 8) * ARITHMETIC * top + EXPONENTIAL


def forward(p, q, k, v, dtype):
    """out and lse [tokens, heads, ..] in 64 bits with their bounds; zeros and 0
    outside the sequences.

    The weights' errors count in the numerators and in their sum; each of these
    rounds once a key, and bf16 weights once more for their product; then the
    quotient and the store."""
    out = torch.zeros(p.tokens, p.heads, p.head_dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.zeros(p.tokens, p.heads, dtype=torch.float64)
    lse_bound = torch.zeros_like(lse)
    q, k, v = q.double(), k.double(), v.double()
    for rows, keys in p.sequences():
        for h in range(p.heads):
            g = p.shared(h)
            w, total, error = _weights(p, q[rows, h], k[keys, g])
            n = keys.stop - keys.start
            y = w @ v[keys, g]
            size = w @ v[keys, g].abs()
            off = 2.0 * error + 2.0 * (n + 8) * ARITHMETIC
            if dtype != torch.float32:
                off = off + ROUNDING[dtype]
            out[rows, h] = y
            bound[rows, h] = off[:, None] * size + ROUNDING[dtype] * (y.abs() + off[:, None] * size)
            lse[rows, h] = total
            finite = torch.where(torch.isfinite(total), total.abs(), 0.0)
            lse_bound[rows, h] = error + (n + 8) * ARITHMETIC + 8 * ARITHMETIC * (finite + 16.0)
    return out, bound, lse, lse_bound


def gradients(p, q, k, v, grad, dtype):
    """Of q, k and v in 64 bits, each with its bound.

    Weights come from the kept log-sum-exp, whose error is a relative one of
    theirs; delta from the kept result, off by its bound times the gradient; the
    slopes are rounded for their products as the weights are."""
    q, k, v, grad = q.double(), k.double(), v.double(), grad.double()
    _, out_bound, _, lse_bound = forward(p, q, k, v, dtype)
    result = [torch.zeros_like(x) for x in (q, k, v)]
    bound = [torch.zeros_like(x) for x in (q, k, v)]
    narrow = ROUNDING[dtype] if dtype != torch.float32 else 0.0
    for rows, keys in p.sequences():
        count, n = rows.stop - rows.start, keys.stop - keys.start
        for h in range(p.heads):
            g = p.shared(h)
            w, lse, error = _weights(p, q[rows, h], k[keys, g])
            d, kh, vh, qh = grad[rows, h], k[keys, g], v[keys, g], q[rows, h]
            off = (2.0 * error + lse_bound[rows, h])[:, None]  # of a weight
            dp = d @ vh.t()
            y = w @ vh
            delta = (d * y).sum(dim=1, keepdim=True)
            slopes = w * (dp - delta)
            delta_off = (d.abs() * (out_bound[rows, h] + (p.head_dim + 2) * ARITHMETIC * y.abs())).sum(1, keepdim=True)
            dp_off = (p.head_dim + 2) * ARITHMETIC * (d.abs() @ vh.abs().t())
            slope_off = w * (1.0 + off) * (dp_off + delta_off) + slopes.abs() * (off + narrow + 4 * ARITHMETIC)
            result[0][rows, h] += p.scale * slopes @ kh
            bound[0][rows, h] += p.scale * (slope_off + (n + 4) * ARITHMETIC * slopes.abs()) @ kh.abs()
            result[1][keys, g] += p.scale * slopes.t() @ qh
            many = (p.heads // p.kv_heads) * count + 4
            bound[1][keys, g] += p.scale * (slope_off + many * ARITHMETIC * slopes.abs()).t() @ qh.abs()
            result[2][keys, g] += w.t() @ d
            bound[2][keys, g] += (w * (off + narrow + many * ARITHMETIC)).t() @ d.abs()
    for x, b in zip(result, bound):
        b += ROUNDING[dtype] * (x.abs() + b)
    return result, bound
