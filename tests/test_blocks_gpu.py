"""The operators together, as a rotary, gated block runs them: eager, captured
into a graph, on another stream, and from several threads."""

from __future__ import annotations

import threading

import pytest
import torch

import blocks_support as support
import cuvit_amd as cuvit
from test_rotary_gpu import ladder

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Block:
    """x += projection(attention(rotary QK norm(QKV(LN x)))); x += down(gated(LN x))
    for images of rows x columns patches and a class token."""

    def __init__(self, dtype, images=3, side=6, heads=3, hidden=128, seed=0):
        g = support.seeded(seed)
        self.dtype, self.images, self.heads, self.hidden = dtype, images, heads, hidden
        self.tokens, self.width = side * side + 1, 64 * heads
        self.rows = images * self.tokens
        width = self.width

        def matrix(n, k):
            return support.normal(g, n, k, scale=k ** -0.5, dtype=dtype).to(DEV)

        self.w = {"qkv": matrix(3 * width, width), "projection": matrix(width, width),
                  "gated": matrix(2 * hidden, width), "down": matrix(width, hidden)}
        self.bias = {name: support.normal(g, w.shape[0], scale=0.1).to(DEV) for name, w in self.w.items()}
        self.gamma = [support.normal(g, 64, mean=1.0, scale=0.2).to(DEV) for _ in range(2)]
        self.one, self.zero = torch.ones(width, device=DEV), torch.zeros(width, device=DEV)
        grid = torch.stack(torch.meshgrid(torch.arange(side), torch.arange(side), indexing="ij"), -1).reshape(-1, 2)
        self.positions = torch.cat([torch.zeros(1, 2), grid.float()]).to(DEV)
        self.frequencies = ladder([16, 16]).to(DEV)
        self.x = support.normal(g, self.rows, width, dtype=dtype).to(DEV)
        self.norm = torch.empty_like(self.x)
        self.qkv = torch.empty(self.rows, 3 * width, dtype=dtype, device=DEV)
        self.context = torch.empty_like(self.x)
        self.hidden_rows = torch.empty(self.rows, hidden, dtype=dtype, device=DEV)
        self.qk = cuvit.qk_norm_problem(images, self.tokens, heads, 64, [16, 16])
        self.gate = cuvit.gated_problem(self.rows, hidden, width, cuvit.GATE_SILU)

    def linear(self, a, name, out, accumulate=False):
        w = self.w[name]
        problem = cuvit.gemm_problem(self.rows, w.shape[0], w.shape[1], cuvit.TRANSPOSED)
        problem.epilogue.accumulate = int(accumulate)
        cuvit.gemm(a, w, self.bias[name], out, problem)

    def run(self, x):
        cuvit.layer_norm(x, self.one, self.zero, self.norm, self.rows, self.width)
        self.linear(self.norm, "qkv", self.qkv)
        cuvit.qk_norm_rotary(self.qkv, *self.gamma, self.positions, self.frequencies, self.qkv, self.qk)
        cuvit.attention(self.qkv, self.context, self.images, self.heads, self.tokens, 64)
        self.linear(self.context, "projection", x, accumulate=True)
        cuvit.layer_norm(x, self.one, self.zero, self.norm, self.rows, self.width)
        cuvit.gated_gemm(self.norm, self.w["gated"], self.bias["gated"], self.hidden_rows, self.gate)
        self.linear(self.hidden_rows, "down", x, accumulate=True)

    def expected(self):
        """In 64 bits on the CPU, with no rounding between the steps."""
        w = {name: t.double().cpu() for name, t in self.w.items()}
        bias = {name: t.double().cpu() for name, t in self.bias.items()}
        x = self.x.double().cpu()

        def norm(t):
            return support.normalise(t, True, 1e-6)[0]

        qkv = (norm(x) @ w["qkv"].t() + bias["qkv"]).reshape(self.images, self.tokens, 3 * self.heads, 64)
        qkv, _ = support.qk_norm(qkv, self.heads, self.heads, False, 1e-6, [g.cpu() for g in self.gamma], [None, None],
                                 (self.positions.cpu(), self.frequencies.cpu(), [16, 16], False))
        q, k, v = (t.transpose(1, 2) for t in qkv.reshape(self.images, self.tokens, 3, self.heads, 64).unbind(2))
        context = torch.softmax(q @ k.transpose(-1, -2) / 8.0, dim=-1) @ v
        x = x + context.transpose(1, 2).reshape(self.rows, self.width) @ w["projection"].t() + bias["projection"]
        z = norm(x) @ w["gated"].t() + bias["gated"]
        hidden = support.activation(0, z[:, :self.hidden]) * z[:, self.hidden:]
        return x + hidden @ w["down"].t() + bias["down"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("images,side,heads", [(1, 1, 3), (3, 6, 3), (2, 14, 6)])
def test_block(dtype, images, side, heads):
    """Each of the eight launches rounds its results once, and what they are
    summed with (fp32: sums of at most 3 * 384 products, 2^-24 of their sizes
    each): eight stages of 2^-8 (bf16) or a generous 2^-15 (fp32) of values that
    stay below 8 after every normalisation."""
    block = Block(dtype, images, side, heads)
    expected = block.expected()
    x = block.x.clone()
    block.run(x)
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -15
    error = (x.cpu().double() - expected).abs()
    assert float(error.max()) <= 8 * unit * float(expected.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(dtype):
    """A graph of the block gives the eager bits on every replay, with eager work
    on the same buffers in between."""
    block = Block(dtype)
    inputs = [support.normal(support.seeded(s), *block.x.shape, dtype=dtype).to(DEV) for s in range(4)]
    eager = []
    for x in inputs:
        x = x.clone()
        block.run(x)
        eager.append(x)
    x = inputs[0].clone()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        block.run(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.run(x)
    for given, wanted in zip(inputs, eager):
        x.copy_(given)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, wanted)
        block.run(given.clone())


def gradients(case, workspace, stream=None):
    qkv, grad, q_gamma, k_gamma, at, turns = case.gpu(case.qkv, case.grad, *case.gamma, case.positions, case.frequencies)
    out = torch.empty_like(grad)
    sums = [torch.empty(qkv.shape[-1], device=DEV) for _ in range(4)]
    torch.cuda.synchronize()

    def run():
        cuvit.qk_norm_rotary_backward(qkv, q_gamma, k_gamma, at, turns, grad, out, case.problem, workspace=workspace,
                                      grad_q_gamma=sums[0], grad_k_gamma=sums[1], grad_q_beta=sums[2],
                                      grad_k_beta=sums[3], stream=stream)
    return run, [out] + sums


def test_backward_captured_and_replayed():
    from test_qk_norm_gpu import Case

    case = Case(torch.bfloat16, 4, 50, 6, 6, 64, [16, 16], beta=True)
    space = torch.empty(cuvit.qk_norm_rotary_workspace(case.problem), dtype=torch.uint8, device=DEV)
    run, results = gradients(case, space)
    run()
    torch.cuda.synchronize()
    wanted = [t.clone() for t in results]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(4):
        space.fill_(255)
        for t in results:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, wanted))
        run()


def test_two_streams_at_once():
    """Launches on two streams, a workspace each, give each alone's bits."""
    from test_qk_norm_gpu import Case

    cases = [Case(torch.float32, 8, 100, 4, 4, 64, [16, 16], beta=True, seed=s) for s in (0, 1)]
    space = [torch.empty(cuvit.qk_norm_rotary_workspace(c.problem), dtype=torch.uint8, device=DEV) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    jobs = [gradients(c, w, s) for c, w, s in zip(cases, space, streams)]
    wanted = []
    for run, results in jobs:
        run()
        torch.cuda.synchronize()
        wanted.append([t.clone() for t in results])
    for _ in range(10):
        for run, _ in jobs:
            run()
    torch.cuda.synchronize()
    for (_, results), alone in zip(jobs, wanted):
        assert all(torch.equal(a, b) for a, b in zip(results, alone))


def test_threads():
    """Threads of one process, a stream and buffers each."""
    wanted, produced, blocks = [], [None] * 4, [Block(torch.bfloat16, seed=s) for s in range(4)]
    for block in blocks:
        x = block.x.clone()
        block.run(x)
        wanted.append(x)
    torch.cuda.synchronize()

    def work(index):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                x = blocks[index].x.clone()
                blocks[index].run(x)
            torch.cuda.current_stream().synchronize()
            produced[index] = x

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(p is not None and torch.equal(p, w) for p, w in zip(produced, wanted))


def test_the_native_module_takes_these_calls():
    block = Block(torch.float32)
    native = cuvit._native_calls
    out, x = torch.empty_like(block.qkv), block.qkv.normal_()
    pre, grad = (torch.randn(block.rows, n * block.hidden, device=DEV) for n in (2, 1))
    space = torch.empty(cuvit.qk_norm_rotary_workspace(block.qk), dtype=torch.uint8, device=DEV)
    rotary = cuvit.rotary_problem(block.images, block.tokens, block.heads, 64, [16, 16])
    sums = torch.empty(64, device=DEV)
    for stream in (None, torch.cuda.Stream(), torch.cuda.current_stream()):
        assert native.rotary(x, block.positions, block.frequencies, out, rotary, stream, None) == 0
        assert native.qk_norm_rotary(x, *block.gamma, block.positions, block.frequencies, out, block.qk, None, None,
                                     stream, None) == 0
        assert native.qk_norm_rotary_backward(x, *block.gamma, block.positions, block.frequencies, x, out, block.qk,
                                              space, sums, None, None, None, stream, None) == 0
        assert native.gated_gemm(block.norm, block.w["gated"], block.bias["gated"], block.hidden_rows, block.gate, pre,
                                 stream, None) == 0
        assert native.gated_backward(pre, grad, pre, block.gate, stream, None) == 0
    torch.cuda.synchronize()
