"""The rotary, QK-norm and gated operators written out in 64 bits, and how far a
kernel may be from them.

The bounds count roundings: u = eps / 2 of the type, 2^-24 for fp32 arithmetic.
"""

from __future__ import annotations

import math

import torch

ARITHMETIC = 2.0 ** -24
ROUNDING = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def normal(generator, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=generator) * scale + mean).to(dtype)


def seeded(seed):
    return torch.Generator().manual_seed(seed)


def angles(positions, frequencies, pairs):
    """[.., tokens, total pairs] in 64 bits."""
    columns, at = [], 0
    for axis, count in enumerate(pairs):
        columns.append(positions.double()[..., axis:axis + 1] * frequencies.double()[at:at + count])
        at += count
    return torch.cat(columns, dim=-1)


def partners(head_dim, pairs, adjacent):
    """Index of each rotated value's first and second partner."""
    total = sum(pairs)
    if adjacent:
        return torch.arange(0, 2 * total, 2), torch.arange(1, 2 * total, 2)
    return torch.arange(total), torch.arange(total, 2 * total)


def rotate(x, positions, frequencies, pairs, adjacent, inverse=False):
    """x [images, tokens, heads, head_dim] in 64 bits."""
    if sum(pairs) == 0:
        return x.clone()
    theta = angles(positions, frequencies, pairs)
    theta = (theta if theta.dim() == 3 else theta[None])[:, :, None, :] * (-1.0 if inverse else 1.0)
    first, second = partners(x.shape[-1], pairs, adjacent)
    out = x.clone()
    out[..., first] = x[..., first] * torch.cos(theta) - x[..., second] * torch.sin(theta)
    out[..., second] = x[..., second] * torch.cos(theta) + x[..., first] * torch.sin(theta)
    return out


def rotation_bound(x, out, pairs, adjacent, dtype):
    """cos and sin are within 2^-22 (the reduced angle's two roundings, 2^-23.3,
    and the series' own), the product and the fused multiply-add round once each:
    (|x| + |y|) (2^-22 + 2^-23) below (|x| + |y|) 2^-21; then the store."""
    first, second = partners(x.shape[-1], pairs, adjacent)
    spread = torch.zeros_like(x)
    both = x[..., first].abs() + x[..., second].abs()
    spread[..., first] = both
    spread[..., second] = both
    stored = ROUNDING[dtype] * out.abs() if dtype != torch.float32 else 0.0
    return spread * 2.0 ** -21 + stored


def normalise(x, layer, epsilon):
    centred = x - x.mean(-1, keepdim=True) if layer else x
    scale = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + epsilon)
    return centred * scale, scale


def by_head(weights, heads, kv_heads, head_dim, missing):
    """[heads + kv_heads, head_dim] in 64 bits from a query and a key row."""
    rows = [torch.full((head_dim,), missing, dtype=torch.float64) if w is None else w.double() for w in weights]
    return torch.cat([rows[0].expand(heads, -1), rows[1].expand(kv_heads, -1)])


def qk_norm(qkv, heads, kv_heads, layer, epsilon, gamma, beta, rotation):
    """The whole packed result in 64 bits, and the normalised, scaled heads
    before the rotation. gamma and beta are (query's, key's), rotation is
    (positions, frequencies, pairs, adjacent)."""
    normed = heads + kv_heads
    head_dim = qkv.shape[-1]
    n, _ = normalise(qkv[:, :, :normed].double(), layer, epsilon)
    y = n * by_head(gamma, heads, kv_heads, head_dim, 1.0) + by_head(beta, heads, kv_heads, head_dim, 0.0)
    return torch.cat([rotate(y, *rotation), qkv[:, :, normed:].double()], dim=2), y


def qk_norm_bound(out, y, dtype):
    """A row's sum of squares is within about 2 * 16 + 6 roundings, its root and
    the factor within half of that and two more; with kLayer the deviations carry
    as much of the row's largest. Both stay below 2^-18 of the row's largest
    scaled value; the rotation adds two such values and its own 2^-20."""
    normed = y.shape[2]
    bound = torch.zeros_like(out)
    bound[:, :, :normed] = 2.0 ** -16.5 * y.abs().amax(-1, keepdim=True)
    if dtype != torch.float32:
        bound[:, :, :normed] += ROUNDING[dtype] * out[:, :, :normed].abs()
    return bound


def qk_norm_gradients(qkv, grad, heads, kv_heads, layer, epsilon, gamma, rotation):
    """The formula's gradients in 64 bits: of qkv, of gamma and beta ([2,
    head_dim], query then key), each with a bound's scale."""
    normed = heads + kv_heads
    head_dim = qkv.shape[-1]
    n, scale = normalise(qkv[:, :, :normed].double(), layer, epsilon)
    d = rotate(grad[:, :, :normed].double(), *rotation, inverse=True)
    g = d * by_head(gamma, heads, kv_heads, head_dim, 1.0)
    along = (g * n).mean(-1, keepdim=True)
    dx = g - n * along
    if layer:
        dx = dx - g.mean(-1, keepdim=True)
    out = torch.cat([dx * scale, grad[:, :, normed:].double()], dim=2)
    # Every term of dx, its largest over the row.
    terms = scale * (g.abs() + g.abs().mean(-1, keepdim=True) + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    size = torch.zeros_like(out)
    size[:, :, :normed] = terms.amax(-1, keepdim=True)
    parts = (slice(0, heads), slice(heads, normed))
    d_gamma = torch.stack([(d * n)[:, :, p].sum((0, 1, 2)) for p in parts])
    d_beta = torch.stack([d[:, :, p].sum((0, 1, 2)) for p in parts])
    size_gamma = torch.stack([(d.abs() * n.abs().amax(-1, keepdim=True))[:, :, p].sum((0, 1, 2)) for p in parts])
    size_beta = torch.stack([d.abs().amax(-1, keepdim=True).expand_as(d)[:, :, p].sum((0, 1, 2)) for p in parts])
    return out, size, d_gamma, size_gamma, d_beta, size_beta


def activation(kind, x):
    if kind == 0:
        return x / (1.0 + torch.exp(-x))
    if kind == 1:
        return 0.5 * x * torch.erfc(-x / math.sqrt(2.0))
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)))


def slope(kind, x):
    if kind == 0:
        s = 1.0 / (1.0 + torch.exp(-x))
        return s + x * s * (1.0 - s)
    if kind == 1:
        return 0.5 * torch.erfc(-x / math.sqrt(2.0)) + x * torch.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)
    u = math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)
    t = torch.tanh(u)
    return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * x ** 2)


def gated(a, w, bias, kind, dtype):
    """The product and its preactivations in 64 bits, each with its bound.

    A sum of k products rounds k times at most in whatever order, u sum|a w| each
    (and the bias once more); a slope is at most 1.13; an activation is within
    2^-20 of its argument's size (the erf form 3.8e-7 of it, the others a few
    roundings of exp2 and the reciprocal)."""
    n = w.shape[0] // 2
    z = a.double() @ w.double().t()
    size = a.double().abs() @ w.double().abs().t()
    if bias is not None:
        z = z + bias.double()
        size = size + bias.double().abs()
    error = (a.shape[1] + 2) * ARITHMETIC * size
    gate, value = z[:, :n], z[:, n:]
    out = activation(kind, gate) * value
    bound = (1.13 * error[:, :n] + 2.0 ** -20 * gate.abs()) * (value.abs() + error[:, n:]) \
        + activation(kind, gate).abs() * error[:, n:] + 2 * ARITHMETIC * out.abs()
    if dtype != torch.float32:
        bound = bound + ROUNDING[dtype] * (out.abs() + bound)
        error = error + ROUNDING[dtype] * (z.abs() + error)
    return out, bound, z, error


def gated_gradient(z, grad, kind, dtype):
    """In 64 bits, with its bound: slopes as the activations within 2^-20 of
    (1 + |gate|), three products of one rounding each."""
    n = z.shape[1] // 2
    gate, value, d = z[:, :n].double(), z[:, n:].double(), grad.double()
    out = torch.cat([d * value * slope(kind, gate), d * activation(kind, gate)], dim=1)
    bound = torch.cat([(d * value).abs() * (1.0 + gate.abs()), d.abs() * gate.abs()], dim=1) * 2.0 ** -19.5
    if dtype != torch.float32:
        bound = bound + ROUNDING[dtype] * (out.abs() + bound)
    return out, bound


def worst(produced, expected, bound):
    """The largest error in units of its bound (0 / 0 is 0)."""
    error = (produced.detach().cpu().double() - expected).abs()
    assert not bool(torch.isnan(error).any()), "NaN where there is a number"
    return float(torch.where(error > 0, error / bound, torch.zeros_like(error)).max()) if error.numel() else 0.0
