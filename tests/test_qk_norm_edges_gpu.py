"""The QK norm's gradients where they depend on what surrounds a head: what an
earlier kernel left in LDS, and another token's turns."""

from __future__ import annotations

import pytest
import torch

import cuvit_amd as cuvit
from test_qk_norm_gpu import DEV, TYPES, Case

pytestmark = pytest.mark.gpu


def leave_nan_in_lds():
    """A rotation of 256 pairs by NaN: 34 KB of NaN turns a workgroup, sixteen
    workgroups for each compute unit."""
    tokens, head_dim = 65536, 512
    x = torch.ones(1, tokens, 1, head_dim, dtype=torch.bfloat16, device=DEV)
    at = torch.ones(tokens, 1, device=DEV)
    turns = torch.full((head_dim // 2,), float("nan"), device=DEV)
    cuvit.rotary(x, at, turns, x, cuvit.rotary_problem(1, tokens, 1, head_dim, [head_dim // 2]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("head_dim,pairs", [(6, [1, 2]), (36, [9, 9]), (64, [11]), (72, [9, 9]), (88, [22]),
                                            (130, [33, 32]), (510, [255])])
def test_gradients_behind_a_broken_rotation(dtype, layer, head_dim, pairs):
    """Pairs that fill no whole run: the turns behind the last one, which nobody
    writes, are in none of a head's sums."""
    case = Case(dtype, 4, 33, 4, 2, head_dim, pairs, False, layer, beta=layer)
    clean = case.forward()
    leave_nan_in_lds()
    case.check_backward()
    leave_nan_in_lds()
    assert torch.equal(case.forward(), clean)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("head_dim,pairs", [(64, [32]), (72, [18]), (510, [249])])
def test_a_broken_position_spoils_its_own_token(dtype, layer, adjacent, head_dim, pairs):
    """Every other token's position is NaN: the ones between them keep their bits
    (a cut run reads into the next token's turns)."""
    case = Case(dtype, 3, 34, 3, 2, head_dim, pairs, adjacent, layer, beta=layer)
    clean, (gradient, _) = case.forward(), case.backward()
    case.positions[1::2] = float("nan")
    spoiled, (other, _) = case.forward(), case.backward()
    assert torch.equal(spoiled[:, ::2], clean[:, ::2]) and torch.equal(other[:, ::2], gradient[:, ::2])
    assert bool(torch.isnan(spoiled[:, 1::2, :5]).any()) and bool(torch.isnan(other[:, 1::2, :5]).any())
