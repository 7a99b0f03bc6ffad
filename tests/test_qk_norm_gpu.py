"""QK norm with rotation and its gradients against 64 bits."""

from __future__ import annotations

import pytest
import torch

import blocks_support as support
import cuvit_amd as cuvit
from test_rotary_gpu import ladder, positions_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16]
EPSILON = 1.0e-6


class Case:
    """Operands of one problem on the CPU, and the calls on the GPU."""

    def __init__(self, dtype, images, tokens, heads, kv_heads, head_dim, pairs, adjacent=False, layer=False, gamma=True,
                 beta=False, seed=0, scale=1.5, mean=0.0):
        g = support.seeded(seed + head_dim + tokens)
        self.heads, self.kv_heads, self.layer, self.pairs, self.adjacent = heads, kv_heads, layer, pairs, adjacent
        self.qkv = support.normal(g, images, tokens, heads + 2 * kv_heads, head_dim, scale=scale, mean=mean, dtype=dtype)
        self.grad = support.normal(g, images, tokens, heads + 2 * kv_heads, head_dim, dtype=dtype)
        self.gamma = [support.normal(g, head_dim, mean=1.0, scale=0.3) if gamma else None for _ in range(2)]
        self.beta = [support.normal(g, head_dim, scale=0.3) if beta else None for _ in range(2)]
        self.positions = positions_of(g, tokens, max(len(pairs), 1))
        self.frequencies = ladder(pairs) if pairs else torch.zeros(1)
        self.problem = cuvit.qk_norm_problem(images, tokens, heads, head_dim, pairs, int(adjacent),
                                             cuvit.NORM_LAYER if layer else cuvit.NORM_RMS, EPSILON, kv_heads)

    def rotation(self):
        return self.positions, self.frequencies, self.pairs, self.adjacent

    def gpu(self, *tensors):
        return [None if t is None else t.to(DEV) for t in tensors]

    def forward(self, qkv=None, out=None):
        qkv = self.qkv.to(DEV) if qkv is None else qkv
        out = torch.full_like(qkv, 7.0) if out is None else out
        q_gamma, k_gamma, q_beta, k_beta, at, turns = self.gpu(*self.gamma, *self.beta, self.positions, self.frequencies)
        cuvit.qk_norm_rotary(qkv, q_gamma, k_gamma, at, turns, out, self.problem, q_beta=q_beta, k_beta=k_beta)
        return out

    def expected(self):
        return support.qk_norm(self.qkv, self.heads, self.kv_heads, self.layer, EPSILON, self.gamma, self.beta,
                               self.rotation())

    def backward(self, wanted=(True, True, True, True), in_place=False):
        qkv, grad = self.gpu(self.qkv, self.grad)
        q_gamma, k_gamma, at, turns = self.gpu(*self.gamma, self.positions, self.frequencies)
        out = grad if in_place else torch.full_like(grad, 7.0)
        sums = [torch.full((qkv.shape[-1],), 7.0, device=DEV) if w else None for w in wanted]
        workspace = None
        if any(wanted):
            workspace = torch.full((cuvit.qk_norm_rotary_workspace(self.problem),), 255, dtype=torch.uint8, device=DEV)
        cuvit.qk_norm_rotary_backward(qkv, q_gamma, k_gamma, at, turns, grad, out, self.problem, workspace=workspace,
                                      grad_q_gamma=sums[0], grad_k_gamma=sums[1], grad_q_beta=sums[2],
                                      grad_k_beta=sums[3])
        return out, sums

    def check_forward(self):
        expected, y = self.expected()
        out = self.forward()
        assert support.worst(out, expected, support.qk_norm_bound(expected, y, self.qkv.dtype)) <= 1.0
        normed = self.heads + self.kv_heads
        assert torch.equal(out[:, :, normed:].cpu(), self.qkv[:, :, normed:])
        return out

    def check_backward(self):
        """A row's factor and n carry 2^-18 as in the forward, a dozen products
        and a sum over the head as much again: 2^-16.5 of a row's largest term.
        The long sums: each term carries 2^-17 of its size, and a lane adds at
        most (images tokens heads / 512 + 1), a workgroup 256 and the join 48
        partial sums, each with one rounding of what is summed."""
        expected, size, d_gamma, size_gamma, d_beta, size_beta = support.qk_norm_gradients(
            self.qkv, self.grad, self.heads, self.kv_heads, self.layer, EPSILON, self.gamma, self.rotation())
        out, sums = self.backward()
        bound = 2.0 ** -16.5 * size
        if self.qkv.dtype != torch.float32:
            bound = bound + support.ROUNDING[self.qkv.dtype] * expected.abs()
        normed = self.heads + self.kv_heads
        assert support.worst(out[:, :, :normed], expected[:, :, :normed], bound[:, :, :normed]) <= 1.0
        assert torch.equal(out[:, :, normed:].cpu(), self.grad[:, :, normed:])
        steps = self.qkv.shape[0] * self.qkv.shape[1] * self.heads / 512 + 305
        unit = 2.0 ** -17 + steps * support.ARITHMETIC
        assert support.worst(torch.stack(sums[:2]), d_gamma, unit * size_gamma) <= 1.0
        assert support.worst(torch.stack(sums[2:]), d_beta, unit * size_beta) <= 1.0
        return out, sums


SIZES = [(2, [1]), (6, [1, 2]), (10, [2, 2]), (16, [4, 4]), (36, [9, 9]), (48, [12, 12]), (64, [16, 16]),
         (64, [8, 12, 12]), (64, [8, 8]), (64, []), (72, [18, 18]), (80, [8, 16, 16]), (88, [44]), (128, [32, 32]),
         (130, [33, 32]), (256, [64, 32]), (512, [128, 128]), (510, [255])]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("head_dim,pairs", SIZES)
def test_forward_head_sizes(dtype, layer, adjacent, head_dim, pairs):
    Case(dtype, 2, 11, 4, 2, head_dim, pairs, adjacent, layer, beta=layer).check_forward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("head_dim,pairs", SIZES)
def test_backward_head_sizes(dtype, layer, adjacent, head_dim, pairs):
    Case(dtype, 2, 11, 4, 2, head_dim, pairs, adjacent, layer, beta=layer).check_backward()


EXTENTS = [(1, 1, 1, 1), (1, 1, 12, 12), (5, 1, 3, 1), (1, 197, 3, 3), (3, 50, 12, 4), (2, 577, 2, 2), (1, 2, 300, 100),
           (1, 3, 1, 130), (40, 30, 1, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("images,tokens,heads,kv_heads", EXTENTS)
def test_extents(dtype, images, tokens, heads, kv_heads):
    for case in (Case(dtype, images, tokens, heads, kv_heads, 64, [16, 16]),
                 Case(dtype, images, tokens, heads, kv_heads, 80, [20, 20], layer=True, gamma=False)):
        case.check_forward()
        case.check_backward()


def test_many_tokens():
    """More groups of tokens than workgroups, in both passes."""
    case = Case(torch.bfloat16, 16, 577, 6, 3, 64, [16, 16], beta=True)
    case.check_forward()
    case.check_backward()


@pytest.mark.parametrize("dtype", TYPES)
def test_in_place_is_the_same(dtype):
    case = Case(dtype, 3, 21, 4, 2, 64, [16, 16], beta=True)
    out = case.forward()
    there = case.qkv.to(DEV)
    case.forward(there, there)
    assert torch.equal(there, out)
    apart, sums = case.backward()
    within, other = case.backward(in_place=True)
    assert torch.equal(apart, within) and all(torch.equal(a, b) for a, b in zip(sums, other))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [64, 72])
def test_alignment_and_neighbours(dtype, width):
    """Off a 16-byte address the same bits, and nothing around them."""
    case = Case(dtype, 2, 9, 3, 3, width, [width // 4, width // 4], beta=True)
    expected = case.forward()
    n = case.qkv.numel()
    for shift in (1, 2, 4):
        source = torch.zeros(n + 8, dtype=dtype, device=DEV)
        source[shift:shift + n] = case.qkv.flatten().to(DEV)
        target = torch.full((n + 8,), 7.0, dtype=dtype, device=DEV)
        case.forward(source[shift:shift + n], target[shift:shift + n])
        # (Another kernel: its runs, so the order of a row's sum, may differ.)
        y = case.expected()[1]
        assert support.worst(target[shift:shift + n].reshape(expected.shape), case.expected()[0],
                             support.qk_norm_bound(case.expected()[0], y, dtype)) <= 1.0
        assert bool((target[:shift] == 7.0).all()) and bool((target[shift + n:] == 7.0).all())


@pytest.mark.parametrize("layer", [False, True])
def test_hard_rows(layer):
    """Zero and constant heads, heads far from zero, tiny and large ones; then
    infinities and NaN, which spoil their own head only."""
    case = Case(torch.float32, 1, 12, 2, 2, 64, [16, 16], layer=layer, beta=True)
    x = case.qkv
    x[0, 0] = 0.0
    x[0, 1] = 3.0
    x[0, 2] += 1000.0
    x[0, 3] *= 1e-18
    x[0, 4] *= 1e15
    x[0, 5, :, 1:] = 0.0
    case.check_forward()
    case.check_backward()
    clean, (gradient, _) = case.forward(), case.backward()
    x[0, 7, 1, 3] = float("inf")
    x[0, 8, 2, 5] = float("nan")
    spoiled, (other, _) = case.forward(), case.backward()
    keep = torch.ones(12, 6, dtype=torch.bool)
    keep[7, 1] = keep[8, 2] = False
    assert torch.equal(spoiled[0][keep], clean[0][keep]) and torch.equal(other[0][keep], gradient[0][keep])
    assert bool(torch.isnan(spoiled[0, 7, 1]).any()) and bool(torch.isnan(spoiled[0, 8, 2]).all())


def test_values_pass_bit_for_bit():
    """NaN payloads, infinities and denormals among the values."""
    case = Case(torch.bfloat16, 1, 5, 2, 2, 64, [16, 16])
    bits = torch.randint(-32768, 32768, (1, 5, 2, 64), generator=support.seeded(1), dtype=torch.int16)
    case.qkv[:, :, 4:] = bits.view(torch.bfloat16)
    case.grad[:, :, 4:] = bits.view(torch.bfloat16)
    assert torch.equal(case.forward()[:, :, 4:].contiguous().view(torch.int16).cpu(), bits)
    assert torch.equal(case.backward()[0][:, :, 4:].contiguous().view(torch.int16).cpu(), bits)


def test_wanted_gradients_only():
    case = Case(torch.float32, 2, 9, 3, 2, 64, [16, 16], layer=True, beta=True)
    out, sums = case.backward()
    for wanted in ((False,) * 4, (True, False, False, False), (False, True, False, True)):
        other, some = case.backward(wanted)
        assert torch.equal(out, other)
        for w, a, b in zip(wanted, sums, some):
            assert (b is None) if not w else torch.equal(a, b)


def test_the_same_bits_again():
    case = Case(torch.bfloat16, 8, 197, 6, 6, 64, [16, 16], beta=True)
    first, sums = case.backward()
    for _ in range(3):
        again, others = case.backward()
        assert torch.equal(first, again) and all(torch.equal(a, b) for a, b in zip(sums, others))


def test_no_tokens_give_zero_gradients():
    sums = [torch.full((64,), 7.0, device=DEV) for _ in range(4)]
    for images, tokens in ((0, 5), (5, 0)):
        problem = cuvit.qk_norm_problem(images, tokens, 2, 64, [16, 16])
        empty = torch.empty(0, device=DEV)
        cuvit.qk_norm_rotary_backward(empty, None, None, empty, empty, empty, empty, problem, grad_q_gamma=sums[0],
                                      grad_k_gamma=sums[1], grad_q_beta=sums[2], grad_k_beta=None)
        assert all(bool((s == 0.0).all()) for s in sums[:3]) and bool((sums[3] == 7.0).all())
        cuvit.qk_norm_rotary(empty, None, None, empty, empty, empty, problem)


def test_gradient_against_differences():
    """The kernel's gradients along a direction against central differences of
    the 64-bit forward. The difference is good to 1e-8 of the values; the
    kernel's sum of N products carries its elements' bounds, added up."""
    case = Case(torch.float32, 1, 5, 2, 2, 16, [4, 4], layer=True, beta=True)
    out, sums = case.backward()
    g = support.seeded(2)
    way = support.normal(g, *case.qkv.shape).double()

    def loss(step, part):
        qkv, gamma, beta = case.qkv.double(), list(case.gamma), list(case.beta)
        if part == "qkv":
            qkv = qkv + step * way
        elif part in (0, 1):
            gamma[part] = gamma[part].double() + step * way[0, 0, 0]
        else:
            beta[part - 2] = beta[part - 2].double() + step * way[0, 0, 0]
        y = support.qk_norm(qkv, 2, 2, True, EPSILON, gamma, beta, case.rotation())[0]
        return float((y * case.grad.double()).sum())

    sizes = support.qk_norm_gradients(case.qkv, case.grad, 2, 2, True, EPSILON, case.gamma, case.rotation())
    for part in ("qkv", 0, 1, 2, 3):
        difference = (loss(1e-5, part) - loss(-1e-5, part)) / 2e-5
        produced = out if part == "qkv" else sums[part]
        along = way if part == "qkv" else way[0, 0, 0]
        size = sizes[1] if part == "qkv" else (sizes[3][part] if part < 2 else sizes[5][part - 2])
        bound = 2.0 ** -15 * float((size * along.abs()).sum()) + 1e-5
        assert abs(float((produced.cpu().double() * along).sum()) - difference) <= bound


def test_refused_tensors():
    case = Case(torch.float32, 2, 5, 3, 3, 64, [16, 16])
    x, at, turns, gamma = case.gpu(case.qkv, case.positions, case.frequencies, case.gamma[0])
    out = torch.full_like(x, 7.0)
    grad = torch.zeros_like(x)
    space = torch.empty(cuvit.qk_norm_rotary_workspace(case.problem), dtype=torch.uint8, device=DEV)
    sums = torch.zeros(64, device=DEV)
    for call, message in [
            (lambda: cuvit.qk_norm_rotary(x[:1].contiguous(), gamma, gamma, at, turns, out, case.problem), "qkv holds 2880"),
            (lambda: cuvit.qk_norm_rotary(x, gamma[:63].contiguous(), gamma, at, turns, out, case.problem), "q_gamma holds 63"),
            (lambda: cuvit.qk_norm_rotary(x, gamma, gamma, at, turns, out, case.problem, q_beta=gamma.double()),
             "q_beta holds torch.float64"),
            (lambda: cuvit.qk_norm_rotary(x, gamma, gamma, None, turns, out, case.problem), "A rotation needs positions"),
            (lambda: cuvit.qk_norm_rotary_backward(x, gamma, gamma, at, turns, grad, out, case.problem,
                                                   grad_q_gamma=sums), "QK norm gradients need a 16-byte aligned workspace"),
            (lambda: cuvit.qk_norm_rotary_backward(x, gamma, gamma, at, turns, grad, out, case.problem,
                                                   workspace=space[:-16], grad_q_gamma=sums), "workspace holds"),
            (lambda: cuvit.qk_norm_rotary_backward(x, gamma, gamma, at, turns, grad, out, case.problem,
                                                   workspace=space, grad_q_gamma=sums[:32]), "grad_q_gamma holds 32"),
            (lambda: cuvit.qk_norm_rotary_backward(x, gamma, gamma, at, turns, grad, x, case.problem),
             "QK norm gradients cannot replace")]:
        with pytest.raises(cuvit.InvalidArgument, match=message):
            call()
    assert bool((out == 7.0).all())
