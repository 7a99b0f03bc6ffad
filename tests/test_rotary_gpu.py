"""The multi-axis rotation against 64 bits: pairings, axes, layouts, head sizes
from one pair on, far positions, and what must stay untouched."""

from __future__ import annotations

import pytest
import torch

import blocks_support as support
import cuvit_amd as cuvit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16]


def ladder(pairs, base=10000.0):
    return torch.cat([base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in pairs]).float()


def positions_of(generator, *shape, low=0, high=40):
    return torch.randint(low, high, shape, generator=generator).float()


def compare(x, positions, pairs, adjacent, inverse=False, frequencies=None, problem=None, out=None):
    """x is [images, tokens, heads, head_dim] on the CPU."""
    frequencies = ladder(pairs) if frequencies is None else frequencies
    images, tokens, heads, head_dim = x.shape
    if problem is None:
        problem = cuvit.rotary_problem(images, tokens, heads, head_dim, pairs, int(adjacent))
        problem.inverse = int(inverse)
        problem.rotation.position_stride = positions[0].numel() if positions.dim() == 3 else 0
    out = torch.empty_like(x, device=DEV) if out is None else out
    cuvit.rotary(x.to(DEV), positions.to(DEV), frequencies.to(DEV), out, problem)
    expected = support.rotate(x.double(), positions, frequencies, pairs, adjacent, inverse)
    bound = support.rotation_bound(x.double(), expected, pairs, adjacent, x.dtype)
    assert support.worst(out, expected, bound) <= 1.0
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("head_dim,pairs", [
    (2, [1]), (6, [1, 1, 1]), (6, [2]), (10, [2, 2]), (16, [4, 4]), (32, [5, 5, 6]), (36, [9, 9]), (48, [12, 12]),
    (64, [16, 16]), (64, [8, 12, 12]), (64, [8, 8]), (64, [0, 3, 2]), (72, [18, 18]), (80, [8, 16, 16]), (88, [22, 22]),
    (104, [52]), (128, [32, 32]), (128, [16]), (256, [64, 64]), (258, [129]), (512, [128, 64, 64]), (510, [200, 55])])
def test_head_sizes(dtype, adjacent, head_dim, pairs):
    g = support.seeded(head_dim + len(pairs))
    x = support.normal(g, 2, 9, 3, head_dim, dtype=dtype)
    compare(x, positions_of(g, 9, len(pairs)), pairs, adjacent)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("images,tokens,heads", [(1, 1, 1), (1, 1, 16), (7, 1, 3), (1, 197, 3), (3, 50, 12), (2, 1025, 2),
                                                 (1, 3, 200), (2, 2, 1025), (65, 31, 1)])
def test_extents(dtype, images, tokens, heads):
    g = support.seeded(images + tokens + heads)
    x = support.normal(g, images, tokens, heads, 64, dtype=dtype)
    compare(x, positions_of(g, images, tokens, 2), [16, 16], False)
    compare(x, positions_of(g, tokens, 2), [16, 16], True, inverse=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_heads_before_tokens_and_gaps(dtype):
    """[images, heads, tokens, head_dim] in, tokens with room between them out:
    the room stays as it was."""
    g = support.seeded(3)
    images, tokens, heads, head_dim, pitch = 3, 21, 5, 64, 5 * 64 + 8
    x = support.normal(g, images, heads, tokens, head_dim, dtype=dtype)
    at = positions_of(g, tokens, 2)
    problem = cuvit.rotary_problem(images, tokens, heads, head_dim, [16, 16])
    problem.input.image, problem.input.token, problem.input.head = heads * tokens * head_dim, head_dim, tokens * head_dim
    problem.output.image, problem.output.token = tokens * pitch, pitch
    out = torch.full((images, tokens, pitch), 7.0, dtype=dtype, device=DEV)
    cuvit.rotary(x.to(DEV), at.to(DEV), ladder([16, 16]).to(DEV), out, problem)
    packed = compare(x.transpose(1, 2).contiguous(), at, [16, 16], False)
    assert torch.equal(out[:, :, :heads * head_dim].reshape(packed.shape), packed)
    assert bool((out[:, :, heads * head_dim:] == 7.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("adjacent", [False, True])
def test_alignment_does_not_change_a_bit(dtype, adjacent):
    """Heads that start off a 16-byte address, and head strides that are odd,
    give the packed result's bits, and their neighbours stay."""
    g = support.seeded(4)
    images, tokens, heads, head_dim = 2, 13, 3, 64
    x = support.normal(g, images, tokens, heads, head_dim, dtype=dtype)
    at = positions_of(g, tokens, 2)
    expected = compare(x, at, [16, 16], adjacent)
    shifted = torch.zeros(x.numel() + 8, dtype=dtype, device=DEV)
    for shift in (1, 2, 4):
        source = shifted[shift:shift + x.numel()]
        source.copy_(x.flatten().to(DEV))
        target = torch.full_like(shifted, 7.0)
        cuvit.rotary(source, at.to(DEV), ladder([16, 16]).to(DEV), target[shift:shift + x.numel()],
                     cuvit.rotary_problem(images, tokens, heads, head_dim, [16, 16], int(adjacent)))
        assert torch.equal(target[shift:shift + x.numel()].reshape(expected.shape), expected)
        assert bool((target[:shift] == 7.0).all()) and bool((target[shift + x.numel():] == 7.0).all())
    problem = cuvit.rotary_problem(images, tokens, heads, head_dim, [16, 16], int(adjacent))
    problem.output.head, problem.output.token, problem.output.image = 65, 3 * 65, tokens * 3 * 65
    spaced = torch.full((images, tokens, heads, 65), 7.0, dtype=dtype, device=DEV)
    cuvit.rotary(x.to(DEV), at.to(DEV), ladder([16, 16]).to(DEV), spaced, problem)
    assert torch.equal(spaced[..., :64], expected) and bool((spaced[..., 64] == 7.0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_in_place_and_back(dtype):
    g = support.seeded(6)
    x = support.normal(g, 2, 33, 4, 64, dtype=dtype)
    at, turns = positions_of(g, 33, 2).to(DEV), ladder([16, 16]).to(DEV)
    expected = compare(x, at.cpu(), [16, 16], True)
    there = x.to(DEV)
    problem = cuvit.rotary_problem(2, 33, 4, 64, [16, 16], cuvit.ROTARY_ADJACENT)
    cuvit.rotary(there, at, turns, there, problem)
    assert torch.equal(there, expected)
    problem.inverse = 1
    cuvit.rotary(there, at, turns, there, problem)
    # Both turns' bounds: a pair's values are within twice (|x| + |y|) (2^-21 + a rounding).
    error = (there.cpu().double() - x.double()).abs().reshape(-1, 2)
    size = x.double().abs().reshape(-1, 2).sum(-1, keepdim=True)
    unit = 2.0 ** -21 + (0.0 if dtype == torch.float32 else support.ROUNDING[dtype])
    assert bool((error <= 3 * unit * size).all())


def test_far_and_broken_positions():
    """Integer, fractional and negative positions up to 2^24 keep the angle's
    fraction: within the bound for any position. Infinity and NaN spoil their own
    token only; a frequency of 0 and position 0 change nothing."""
    g = support.seeded(8)
    x = support.normal(g, 1, 64, 2, 64)
    at = torch.cat([positions_of(g, 16, 2, low=2 ** 23, high=2 ** 24), -positions_of(g, 16, 2, low=1000, high=10 ** 6),
                    torch.rand(16, 2, generator=g) * 1000, torch.rand(16, 2, generator=g) * 1e-6])
    for adjacent in (False, True):
        compare(x, at, [16, 16], adjacent)
        compare(x, at, [32, 0], adjacent, frequencies=torch.rand(32, generator=g) * 30 - 15)
        still = compare(x, torch.zeros(64, 2), [16, 16], adjacent)
        assert torch.equal(still.cpu(), x)
        broken = at.clone()
        broken[5, 0], broken[6, 1] = float("inf"), float("nan")
        whole, parts = (torch.empty_like(x, device=DEV) for _ in range(2))
        problem = cuvit.rotary_problem(1, 64, 2, 64, [16, 16], int(adjacent))
        cuvit.rotary(x.to(DEV), at.to(DEV), ladder([16, 16]).to(DEV), whole, problem)
        cuvit.rotary(x.to(DEV), broken.to(DEV), ladder([16, 16]).to(DEV), parts, problem)
        same = torch.ones(64, dtype=torch.bool)
        same[5:7] = False
        assert torch.equal(parts[:, same], whole[:, same])
        assert bool(torch.isnan(parts[:, 5]).any()) and not bool(torch.isnan(parts[:, 5]).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("head_dim,pairs", [(64, [8, 8]), (72, [10, 9]), (64, [5, 6])])
def test_the_unrotated_rest_keeps_its_bits(dtype, adjacent, head_dim, pairs):
    g = support.seeded(9)
    x = support.normal(g, 1, 20, 3, head_dim, dtype=dtype)
    rest = x[..., 2 * sum(pairs):]
    rest[..., 0::3] = float("inf")
    rest[..., 1::3] = float("-inf")
    rest[..., 2::3] = 3e38
    out = torch.empty_like(x, device=DEV)
    cuvit.rotary(x.to(DEV), positions_of(g, 20, 2).to(DEV), ladder(pairs).to(DEV), out,
                 cuvit.rotary_problem(1, 20, 3, head_dim, pairs, int(adjacent)))
    assert torch.equal(out[..., 2 * sum(pairs):].cpu(), rest)
    assert bool(torch.isfinite(out[..., :2 * sum(pairs)]).all())


def test_no_axes_copy():
    x = torch.randn(2, 7, 3, 18).to(DEV)
    out = torch.empty_like(x)
    cuvit.rotary(x, None, None, out, cuvit.rotary_problem(2, 7, 3, 18, []))
    assert torch.equal(out, x)


def test_an_image_alone_gives_the_same_bits():
    g = support.seeded(10)
    x = support.normal(g, 6, 197, 3, 64, dtype=torch.bfloat16).to(DEV)
    at, turns = positions_of(g, 197, 2).to(DEV), ladder([16, 16]).to(DEV)
    whole, alone = torch.empty_like(x), torch.empty_like(x)
    cuvit.rotary(x, at, turns, whole, cuvit.rotary_problem(6, 197, 3, 64, [16, 16]))
    for i in range(6):
        cuvit.rotary(x[i], at, turns, alone[i], cuvit.rotary_problem(1, 197, 3, 64, [16, 16]))
    assert torch.equal(whole, alone)


def test_refused_tensors():
    x, at, turns = torch.zeros(2, 5, 3, 64, device=DEV), torch.zeros(5, 2, device=DEV), torch.zeros(32, device=DEV)
    out = torch.full_like(x, 7.0)
    problem = cuvit.rotary_problem(2, 5, 3, 64, [16, 16])
    for arguments, message in [
            ((x[:1].contiguous(), at, turns, out), "x holds 960 elements"),
            ((x, at[:4].contiguous(), turns, out), "positions holds 8"),
            ((x, at, turns[:31].contiguous(), out), "frequencies holds 31"),
            ((x, at.double(), turns, out), "positions holds torch.float64"),
            ((x, at, turns, out.bfloat16()), "out holds torch.bfloat16"),
            ((x, at, turns, out.transpose(1, 2)), "out is not contiguous"),
            ((x, at.cpu(), turns, out), "positions is not a GPU tensor")]:
        with pytest.raises(cuvit.InvalidArgument, match=message):
            cuvit.rotary(*arguments, problem)
    problem.rotation.position_stride = 10
    with pytest.raises(cuvit.InvalidArgument, match="positions holds 10 elements; the launch touches 20"):
        cuvit.rotary(x, at, turns, out, problem)
    assert bool((out == 7.0).all())


def test_offsets_past_32_bits():
    """Two images 2^31 elements apart in one bf16 buffer (8 GiB)."""
    g = support.seeded(11)
    x = support.normal(g, 2, 4, 3, 64, dtype=torch.bfloat16)
    at = positions_of(g, 4, 2)
    far = torch.empty(2 ** 31 + 8192, dtype=torch.bfloat16, device=DEV)
    problem = cuvit.rotary_problem(2, 4, 3, 64, [16, 16])
    problem.input.image = problem.output.image = 2 ** 31 + 64
    for i in range(2):
        far[i * (2 ** 31 + 64):][:x[i].numel()] = x[i].flatten().to(DEV)
    cuvit.rotary(far, at.to(DEV), ladder([16, 16]).to(DEV), far, problem)
    expected = compare(x, at, [16, 16], False)
    for i in range(2):
        assert torch.equal(far[i * (2 ** 31 + 64):][:x[i].numel()].reshape(x[i].shape), expected[i])


def test_more_tokens_than_workgroups():
    """2^24 tokens of more heads than a workgroup has teams for (40 GB in place):
    each head as if it were the only one."""
    tokens, heads = 2 ** 24 + 5, 600
    at = (torch.arange(tokens, device=DEV) % 10007).float()[:, None]
    turns = ladder([1]).to(DEV)
    alone = torch.ones(1, tokens, 1, 2, dtype=torch.bfloat16, device=DEV)
    cuvit.rotary(alone, at, turns, alone, cuvit.rotary_problem(1, tokens, 1, 2, [1]))
    x = torch.ones(1, tokens, heads, 2, dtype=torch.bfloat16, device=DEV)
    cuvit.rotary(x, at, turns, x, cuvit.rotary_problem(1, tokens, heads, 2, [1]))
    for first in range(0, tokens, 2 ** 20):
        part = slice(first, min(first + 2 ** 20, tokens))
        assert bool((x[:, part] == alone[:, part]).all()), first
