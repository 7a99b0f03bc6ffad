"""A block on packed images of different sizes, forwards and backwards, as a training
step runs it: projection, QK norm and rotation in place, packed attention, gated MLP with
codes kept, and the gradients of each. Every stage is held to its formula on what the
stage before it gave, and the captured step to the eager one's bits."""

from __future__ import annotations

import math

import pytest
import torch

import blocks_support as blocks
from blocks_support import normal, seeded, worst
from packed_support import Packed, forward, gradients
from test_gated_checkpoint_gpu import check_codes, values

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, HEAD_DIM, EMBED, HIDDEN = 6, 2, 32, 192, 512
LENGTHS = [50, 197, 1, 65]
PAIRS = [8, 8]


class Step:
    def __init__(self, cuvit, device, dtype, causal):
        self.cuvit = cuvit
        self.p = Packed(LENGTHS, HEADS, HEAD_DIM, kv_heads=KV_HEADS, causal=causal, spare=0)
        tokens, slots = self.p.tokens, HEADS + 2 * KV_HEADS
        generator = seeded(77)

        def to(*shape, scale=1.0, kind=dtype, mean=0.0):
            return normal(generator, *shape, scale=scale, dtype=kind, mean=mean).to(device)

        self.x = to(tokens, EMBED)
        self.w_qkv = to(slots * HEAD_DIM, EMBED, scale=1.0 / math.sqrt(EMBED))
        self.gamma = [to(HEAD_DIM, kind=torch.float32, scale=0.2, mean=1.0) for _ in range(2)]
        self.positions = torch.cat([torch.stack([torch.arange(n) // 14, torch.arange(n) % 14], dim=1).float()
                                    for n in LENGTHS]).to(device)
        self.frequencies = torch.cat([10000.0 ** (-torch.arange(n) / n) for n in PAIRS]).to(device)
        self.w_gated = to(2 * HIDDEN, EMBED, scale=1.0 / math.sqrt(EMBED))
        self.grad_context = to(tokens, HEADS, HEAD_DIM)
        self.grad_hidden = to(tokens, HIDDEN)
        self.starts = torch.tensor(self.p.starts, dtype=torch.int32, device=device)

        def room(*shape, kind=dtype):
            return torch.zeros(*shape, dtype=kind, device=device)

        self.qkv, self.normed, self.grad_qkv, self.grad_projection = (room(tokens, slots, HEAD_DIM) for _ in range(4))
        self.context, self.lse = room(tokens, HEADS, HEAD_DIM), room(tokens, HEADS, kind=torch.float32)
        self.hidden, self.again, self.grad_pre = room(tokens, HIDDEN), room(tokens, HIDDEN), room(tokens, 2 * HIDDEN)
        self.grad_gamma = [room(HEAD_DIM, kind=torch.float32) for _ in range(2)]
        self.gated = cuvit.gated_problem(tokens, HIDDEN, EMBED)
        self.codes = room(tokens, 2 * HIDDEN, kind=torch.float8_e4m3fn)
        self.scales = torch.zeros(cuvit.gated_checkpoint_scales(self.gated), dtype=torch.uint8,
                                  device=device).view(torch.float8_e8m0fnu)
        self.norm = cuvit.qk_norm_problem(1, tokens, HEADS, HEAD_DIM, PAIRS, kv_heads=KV_HEADS)
        self.attention = cuvit.packed_attention_problem(len(LENGTHS), tokens, HEADS, HEAD_DIM, kv_heads=KV_HEADS,
                                                        causal=causal, projection=True)
        size = max(cuvit.packed_attention_workspace(self.attention),
                   cuvit.packed_attention_backward_workspace(self.attention), cuvit.qk_norm_rotary_workspace(self.norm))
        self.workspace = room(size, kind=torch.uint8)  # one stream: its calls follow one another

    def run(self):
        c, tokens = self.cuvit, self.p.tokens
        c.gemm(self.x, self.w_qkv, None, self.qkv, c.gemm_problem(tokens, self.w_qkv.shape[0], EMBED, c.TRANSPOSED))
        c.qk_norm_rotary(self.qkv, *self.gamma, self.positions, self.frequencies, self.normed, self.norm)
        c.packed_attention(self.normed, None, None, self.starts, self.context, self.attention, lse=self.lse,
                           workspace=self.workspace)
        c.gated_checkpoint_gemm(self.context, self.w_gated, None, self.hidden, self.codes, self.scales, self.gated)
        c.gated_checkpoint_backward(self.codes, self.scales, self.grad_hidden, self.grad_pre, self.gated,
                                    hidden=self.again)
        c.packed_attention_backward(self.normed, None, None, self.starts, self.context, self.lse, self.grad_context,
                                    self.grad_qkv, None, None, self.attention, workspace=self.workspace)
        c.qk_norm_rotary_backward(self.qkv, *self.gamma, self.positions, self.frequencies, self.grad_qkv,
                                  self.grad_projection, self.norm, workspace=self.workspace,
                                  grad_q_gamma=self.grad_gamma[0], grad_k_gamma=self.grad_gamma[1])

    def results(self):
        return [self.qkv, self.normed, self.context, self.lse, self.hidden, self.codes.view(torch.uint8),
                self.scales.view(torch.uint8), self.grad_pre, self.again, self.grad_qkv, self.grad_projection,
                *self.grad_gamma]


@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_step(cuvit, device, dtype, causal):
    s = Step(cuvit, device, dtype, causal)
    s.run()
    torch.cuda.synchronize()
    parts = [HEADS, KV_HEADS, KV_HEADS]
    q, k, v = s.normed.cpu().split(parts, dim=1)
    expected, bound, lse, lse_bound = forward(s.p, q, k, v, dtype)
    assert worst(s.context, expected, bound) <= 1.0 and worst(s.lse, lse, lse_bound) <= 1.0
    context = s.context.cpu().reshape(s.p.tokens, EMBED)
    expected, bound, z, error = blocks.gated(context, s.w_gated.cpu(), None, 0, dtype)
    assert worst(s.hidden, expected, bound) <= 1.0
    if dtype != torch.float32:
        error = blocks.gated(context.float(), s.w_gated.cpu().float(), None, 0, torch.float32)[3]
    check_codes(s.codes, s.scales, z, error, HIDDEN)
    expected, bound = blocks.gated_gradient(values(s.codes, s.scales, HIDDEN), s.grad_hidden.cpu(), 0, dtype)
    assert worst(s.grad_pre, expected, bound) <= 1.0
    expected, bounds = gradients(s.p, q, k, v, s.grad_context.cpu(), dtype)
    for produced, e, b in zip(s.grad_qkv.cpu().split(parts, dim=1), expected, bounds):
        assert worst(produced, e, b) <= 1.0
    rotation = (s.positions.cpu(), s.frequencies.cpu(), PAIRS, False)
    out, size, *_ = blocks.qk_norm_gradients(s.qkv.cpu()[None], s.grad_qkv.cpu()[None], HEADS, KV_HEADS, False, 1e-6,
                                             [g.cpu() for g in s.gamma], rotation)
    # (The norm's gradients are held to tighter bounds by tests of their own.)
    off = 2.0 ** -14 * size + blocks.ROUNDING[dtype] * out.abs()
    assert worst(s.grad_projection, out[0], off[0]) <= 1.0

    eager = [x.clone() for x in s.results()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    for _ in range(3):
        for x in s.results():
            x.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(s.results(), eager))
