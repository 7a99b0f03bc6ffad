"""Gated products that keep 8-bit codes of their preactivations, and the gradient from
them, against their definitions in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from blocks_support import ROUNDING, activation, gated, gated_gradient, normal, seeded, worst

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
GROUP = 32


def kept(p, cuvit, device, ld=None):
    codes = torch.full((p.m, ld or 2 * p.n), 8.0, device=device).to(torch.float8_e4m3fn)
    scales = torch.full((cuvit.gated_checkpoint_scales(p),), 4.0, device=device).to(torch.float8_e8m0fnu)
    return codes, scales


def values(codes, scales, n):
    """The preactivations that codes stand for, in 64 bits on the CPU."""
    m = codes.shape[0]
    powers = scales.cpu().float().double().reshape(m, 2, -1).repeat_interleave(GROUP, dim=2)[:, :, :n]
    return codes.cpu()[:, :2 * n].float().double() * powers.reshape(m, 2 * n)


def groups_of(z, n):
    return torch.nn.functional.pad(z.reshape(z.shape[0], 2, n), (0, -n % GROUP)).reshape(z.shape[0], 2, -1, GROUP)


def least_scale(largest):
    """The least power of two from 2^-117 on that keeps `largest` within 448 of it."""
    mantissa, exponent = torch.frexp(largest)  # (of 0 it says 2^0)
    return torch.exp2(torch.where(largest > 0, exponent - 9 + (mantissa > 0.875), -117).clamp(min=-117).double())


def check_codes(codes, scales, z, error, n):
    """Every scale is the least for a largest value within `error` of the exact one,
    and every value within that error and half a step: 2^-4 of it, or 2^-10 of the
    scale."""
    size, off = groups_of(z.abs(), n), groups_of(error, n)
    low, high = (size - off).clamp(min=0.0).amax(-1), (size + off).amax(-1)
    powers = scales.cpu().float().double().reshape(low.shape)
    assert bool(((powers == least_scale(low)) | (powers == least_scale(high))).all())
    spread = powers.repeat_interleave(GROUP, dim=2)[:, :, :n].reshape(z.shape)
    bound = error + torch.maximum(2.0 ** -4 * (z.abs() + error), 2.0 ** -10 * spread)
    assert worst(values(codes, scales, n), z, bound) <= 1.0


# Every kernel and tile: few rows, small and large tiles of the ring, and rows that are
# no whole chunks.
SIZES = [(1, 17, 24), (5, 32, 8), (40, 96, 64), (65, 33, 40), (66, 70, 37), (100, 683, 96), (197, 512, 192),
         (394, 2048, 768), (788, 1365, 512), (1576, 2048, 128), (3152, 2048, 72), (4616, 2048, 64),
         (3152, 2048, 71), (2308, 1024, 33), (7000, 512, 64)]


@TYPES
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_and_codes(cuvit, device, dtype, m, n, k):
    kind = (m + n) % 3
    generator = seeded(m + n)
    a = normal(generator, m, k, dtype=dtype)
    w = normal(generator, 2 * n, k, scale=1.0 / math.sqrt(k), dtype=dtype)
    bias = normal(generator, 2 * n, scale=0.1) if m % 2 == 0 else None
    p = cuvit.gated_problem(m, n, k, kind)
    out = torch.zeros(m, n, dtype=dtype, device=device)
    codes, scales = kept(p, cuvit, device)
    ga, gw, gb = a.to(device), w.to(device), bias.to(device) if bias is not None else None
    cuvit.gated_checkpoint_gemm(ga, gw, gb, out, codes, scales, p)
    expected, bound, z, error = (x.cpu() for x in gated(ga, gw, gb, kind, dtype))
    if dtype != torch.float32:  # codes come from the sums, not from stored preactivations
        error = gated(ga.float(), gw.float(), gb, kind, torch.float32)[3].cpu()
    assert worst(out, expected, bound) <= 1.0
    check_codes(codes, scales, z, error, n)
    if m > 64:  # the same sums as the product that stores its preactivations
        plain, pre = torch.zeros_like(out), torch.zeros(m, 2 * n, dtype=dtype, device=device)
        cuvit.gated_gemm(ga, gw, gb, plain, p, preactivations=pre)
        assert torch.equal(plain, out)


@TYPES
@pytest.mark.parametrize("m,n,k", [(3, 96, 16), (100, 1000, 16), (100, 1000, 13), (3200, 2048, 16), (300, 77, 16)])
def test_codes_of_known_values(cuvit, device, dtype, m, n, k):
    """Preactivations that are the bias: sizes from the smallest to the largest floats,
    ties, borders of a scale, zeros, infinities and NaN, each code bit for bit."""
    generator = seeded(n)
    bias = normal(generator, 2 * n) * torch.exp2(torch.randint(-60, 60, (2 * n,), generator=generator).float())
    for at, value in enumerate([0.0, -0.0, 3.0e38, -3.4e38, 1e-45, 2.0 ** -126, 448.0, 464.0, 449.0, 1.75, 1.7500001]):
        bias[(7 * at) % n] = value
    bias[n:n + 32] = 2.0 ** -130 * torch.arange(32)                   # a group below every scale
    if n >= 96:
        bias[32:64] = torch.arange(32) / 16.0 + 1.0 / 32.0            # ties
        bias[64] = math.inf
        bias[65] = math.nan
        bias[n + 32:n + 64] = -math.inf                               # nothing finite
    a = torch.zeros(m, k, dtype=dtype, device=device)
    w = torch.ones(2 * n, k, dtype=dtype, device=device)
    p = cuvit.gated_problem(m, n, k)
    codes, scales = kept(p, cuvit, device)
    out = torch.zeros(m, n, dtype=dtype, device=device)
    cuvit.gated_checkpoint_gemm(a, w, bias.to(device), out, codes, scales, p)
    finite = torch.where(torch.isfinite(bias), bias.double(), 0.0)
    powers = least_scale(groups_of(finite[None], n).abs().amax(-1))
    assert torch.equal(scales.cpu().float().double().reshape(m, 2, -1), powers.expand(m, -1, -1))
    # (Products of 0 are added: a bias of -0 gives 0.)
    scaled = (bias.double() + 0.0) / powers.repeat_interleave(GROUP, dim=2)[:, :, :n].reshape(2 * n)
    expected = torch.where(torch.isfinite(bias), scaled, math.nan).float().to(torch.float8_e4m3fn)
    produced = codes.cpu().float()
    assert bool((torch.isnan(produced) == torch.isnan(expected.float())).all())
    known = ~torch.isnan(expected.float())
    assert torch.equal(codes.cpu().view(torch.uint8)[:, known],
                       expected.view(torch.uint8)[known].expand(m, -1))


@TYPES
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("m,n", [(1, 1), (3, 31), (7, 33), (197, 683), (65, 2048), (3152, 1365)])
def test_gradient_and_product_from_codes(cuvit, device, dtype, kind, m, n):
    generator = seeded(m * n + kind)
    p = cuvit.gated_problem(m, n, 1, kind)
    codes = (normal(generator, m, 2 * n) * 100.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    scales = torch.randint(118, 124, (cuvit.gated_checkpoint_scales(p),), generator=generator).to(torch.uint8)
    scales = scales.view(torch.float8_e8m0fnu)
    z = values(codes, scales, n)
    grad = normal(generator, m, n, dtype=dtype)
    results = []
    for hidden in (torch.zeros(m, n, dtype=dtype, device=device), None):
        to = torch.zeros(m, 2 * n, dtype=dtype, device=device)
        cuvit.gated_checkpoint_backward(codes.to(device), scales.to(device), grad.to(device), to, p, hidden=hidden)
        results.append(to)
        if hidden is not None:
            again = hidden
    expected, bound = gated_gradient(z, grad, kind, dtype)
    assert worst(results[0], expected, bound) <= 1.0
    assert torch.equal(results[0], results[1])
    product = activation(kind, z[:, :n]) * z[:, n:]
    # (An activation is within 2^-20 of its argument's size; the product rounds once.)
    bound = z[:, :n].abs() * z[:, n:].abs() * 2.0 ** -19.5
    bound = bound + ROUNDING[dtype] * (product.abs() + bound)
    assert worst(again, product, bound) <= 1.0
    same = grad.to(device)
    to = torch.zeros(m, 2 * n, dtype=dtype, device=device)
    cuvit.gated_checkpoint_backward(codes.to(device), scales.to(device), same, to, p, hidden=same)
    assert torch.equal(same, again) and torch.equal(to, results[0])


@TYPES
@pytest.mark.parametrize("m,n,k", [(70, 40, 24), (300, 129, 33), (200, 512, 64)])
def test_leading_dimensions(cuvit, device, dtype, m, n, k):
    """Rows further apart: what lies between them stays."""
    generator = seeded(n)
    p = cuvit.gated_problem(m, n, k)
    p.lda, p.ldb, p.ldc, p.ld_preactivations = k + 8, k + 16, n + 3, 2 * n + 5
    a = normal(generator, m, k + 8, dtype=dtype).to(device)
    w = normal(generator, 2 * n, k + 16, scale=1.0 / math.sqrt(k), dtype=dtype).to(device)
    out = torch.full((m, n + 3), 7.0, dtype=dtype, device=device)
    codes, scales = kept(p, cuvit, device, 2 * n + 5)
    cuvit.gated_checkpoint_gemm(a, w, None, out, codes, scales, p)
    plain = cuvit.gated_problem(m, n, k)
    plain_out = torch.zeros(m, n, dtype=dtype, device=device)
    plain_codes, plain_scales = kept(plain, cuvit, device)
    cuvit.gated_checkpoint_gemm(a[:, :k].contiguous(), w[:, :k].contiguous(), None, plain_out, plain_codes,
                                plain_scales, plain)
    assert torch.equal(out[:, :n], plain_out) and bool((out[:, n:] == 7.0).all())
    assert torch.equal(codes[:, :2 * n].view(torch.uint8), plain_codes.view(torch.uint8))
    assert torch.equal(scales.view(torch.uint8), plain_scales.view(torch.uint8))
    assert bool((codes[:, 2 * n:].float() == 8.0).all())
    grad = normal(generator, m, n + 3, dtype=dtype).to(device)
    to = torch.full((m, 2 * n + 5), 7.0, dtype=dtype, device=device)
    hidden = torch.full((m, n + 3), 7.0, dtype=dtype, device=device)
    cuvit.gated_checkpoint_backward(codes, scales, grad, to, p, hidden=hidden)
    plain_to = torch.zeros(m, 2 * n, dtype=dtype, device=device)
    plain_hidden = torch.zeros(m, n, dtype=dtype, device=device)
    cuvit.gated_checkpoint_backward(plain_codes, plain_scales, grad[:, :n].contiguous(), plain_to, plain,
                                    hidden=plain_hidden)
    assert torch.equal(to[:, :2 * n], plain_to) and bool((to[:, 2 * n:] == 7.0).all())
    assert torch.equal(hidden[:, :n], plain_hidden) and bool((hidden[:, n:] == 7.0).all())


@TYPES
def test_nan_codes_stay(cuvit, device, dtype):
    p = cuvit.gated_problem(1, 64, 1)
    codes = torch.ones(1, 128).to(torch.float8_e4m3fn)
    codes.view(torch.uint8)[0, 5] = 0x7F
    codes.view(torch.uint8)[0, 70] = 0xFF
    scales = torch.ones(4).to(torch.float8_e8m0fnu)
    to = torch.zeros(1, 128, dtype=dtype, device=device)
    hidden = torch.zeros(1, 64, dtype=dtype, device=device)
    cuvit.gated_checkpoint_backward(codes.to(device), scales.to(device), torch.ones(1, 64, dtype=dtype, device=device),
                                    to, p, hidden=hidden)
    bad = torch.isnan(to.cpu()[0])
    assert sorted(torch.nonzero(bad)[:, 0].tolist()) == [5, 6, 69]
    assert sorted(torch.nonzero(torch.isnan(hidden.cpu()[0]))[:, 0].tolist()) == [5, 6]


def test_more_codes_than_32_bits_count(cuvit, device):
    m, n, k = 530_000, 4096, 8
    p = cuvit.gated_problem(m, n, k)
    a = torch.zeros(m, k, dtype=torch.bfloat16, device=device)
    generator = seeded(3)
    a[-3:] = normal(generator, 3, k, dtype=torch.bfloat16).to(device)
    w = normal(generator, 2 * n, k, scale=0.3, dtype=torch.bfloat16).to(device)
    out = torch.zeros(m, n, dtype=torch.bfloat16, device=device)
    codes, scales = kept(cuvit.gated_problem(1, 1, 1), cuvit, device)
    codes = torch.empty(m, 2 * n, dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty(m, 2 * (n // GROUP), dtype=torch.float8_e8m0fnu, device=device)
    cuvit.gated_checkpoint_gemm(a, w, None, out, codes, scales, p)
    z = a[-3:].cpu().double() @ w.cpu().double().t()
    error = (k + 2) * 2.0 ** -24 * (a[-3:].cpu().double().abs() @ w.cpu().double().t().abs())
    check_codes(codes[-3:], scales[-3:].reshape(-1), z, error, n)
    grad = torch.ones(m, n, dtype=torch.bfloat16, device=device)
    to = torch.zeros(m, 2 * n, dtype=torch.bfloat16, device=device)
    cuvit.gated_checkpoint_backward(codes, scales, grad, to, p, hidden=grad)
    expected, bound = gated_gradient(values(codes[-3:], scales[-3:].reshape(-1), n), torch.ones(3, n), 0, torch.bfloat16)
    assert worst(to[-3:], expected, bound) <= 1.0


@TYPES
def test_captured(cuvit, device, dtype):
    m, n, k = 197, 512, 192
    generator = seeded(9)
    p = cuvit.gated_problem(m, n, k)
    a, w = normal(generator, m, k, dtype=dtype).to(device), normal(generator, 2 * n, k, scale=0.1, dtype=dtype).to(device)
    grad = normal(generator, m, n, dtype=dtype).to(device)

    def buffers():
        return (torch.zeros(m, n, dtype=dtype, device=device), *kept(p, cuvit, device),
                torch.zeros(m, 2 * n, dtype=dtype, device=device), torch.zeros(m, n, dtype=dtype, device=device))

    def run(out, codes, scales, to, hidden):
        cuvit.gated_checkpoint_gemm(a, w, None, out, codes, scales, p)
        cuvit.gated_checkpoint_backward(codes, scales, grad, to, p, hidden=hidden)

    captured = buffers()
    graph = torch.cuda.CUDAGraph()
    run(*captured)  # (LDS is opted in to before)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        run(*captured)
    for turn in range(3):
        a.copy_(normal(generator, m, k, dtype=dtype))
        eager = buffers()
        run(*eager)
        for x in captured:
            x.view(torch.uint8).fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(captured, eager))
