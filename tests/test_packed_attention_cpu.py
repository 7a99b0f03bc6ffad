"""What attention over packed sequences refuses, its workspaces, and the 64-bit
formula that the GPU tests hold it to, against differences."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import cuvit_amd as cuvit
from blocks_support import normal, seeded
from packed_support import Packed, forward, gradients

INT_MAX = 2 ** 31 - 1
ADDRESS = 1 << 20  # never read: every call here is refused, or has nothing to do


def problem(**fields):
    p = cuvit.packed_attention_problem(2, 10, 4, 64, kv_heads=2)
    for name, value in fields.items():
        target = p
        *path, last = name.split("__")
        for part in path:
            target = getattr(target, part)
        setattr(target, last, value)
    return p


def forward_call(lib, p, q=ADDRESS, k=ADDRESS, v=ADDRESS, starts=ADDRESS, kv_starts=None, kv_lengths=None,
                 out=ADDRESS * 2, lse=None, workspace=None, nbytes=0, bf16=True):
    fn = lib.cuvit_packed_attention_bf16 if bf16 else lib.cuvit_packed_attention_f32
    return fn(q, k, v, starts, kv_starts, kv_lengths, out, lse, workspace, nbytes,
              ctypes.byref(p) if p is not None else None, None)


def backward_call(lib, p, q=ADDRESS, k=ADDRESS, v=ADDRESS, starts=ADDRESS, kv_starts=None, out=ADDRESS, lse=ADDRESS,
                  grad_out=ADDRESS, grad_q=2 * ADDRESS, grad_k=2 * ADDRESS, grad_v=2 * ADDRESS, workspace=ADDRESS,
                  nbytes=1 << 40, bf16=True):
    fn = lib.cuvit_packed_attention_backward_bf16 if bf16 else lib.cuvit_packed_attention_backward_f32
    return fn(q, k, v, starts, kv_starts, None, out, lse, grad_out, grad_q, grad_k, grad_v, workspace, nbytes,
              ctypes.byref(p) if p is not None else None, None)


CALLS = pytest.mark.parametrize("call", [forward_call, backward_call], ids=["forward", "backward"])


@CALLS
@pytest.mark.parametrize("fields", [dict(sequences=0), dict(heads=0), dict(head_dim=0), dict(tokens=0, kv_tokens=0)])
def test_nothing_to_do(lib, call, fields):
    nothing = {name: None for name in ("q", "k", "v", "starts", "out")}
    assert call(lib, problem(**fields), **nothing) == cuvit.OK


INVALID = [
    dict(sequences=-1), dict(tokens=-1), dict(kv_tokens=-1), dict(heads=-1), dict(head_dim=-8), dict(kv_heads=0),
    dict(kv_heads=-2), dict(kv_heads=3), dict(kv_heads=8), dict(head_dim=60), dict(head_dim=264), dict(head_dim=2),
    dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(scale=1e-45),
    dict(q__token=-256), dict(k__head=-64), dict(v__token=68), dict(out__head=4), dict(q__token=56), dict(k__token=32),
]


@CALLS
@pytest.mark.parametrize("fields", INVALID, ids=[str(f) for f in INVALID])
def test_invalid_problems(lib, call, fields):
    assert call(lib, problem(**fields)) == cuvit.ERROR_INVALID_ARGUMENT
    assert lib.cuvit_last_error()


@pytest.mark.parametrize("fields", [dict(out__token=128), dict(out__token=64, out__head=64),
                                    dict(out__token=256, out__head=128), dict(out__token=256, out__head=32)])
def test_overlapping_results(lib, fields):
    assert forward_call(lib, problem(**fields)) == cuvit.ERROR_INVALID_ARGUMENT
    assert b"overlap" in lib.cuvit_last_error()


@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_overlapping_gradients(lib, name):
    assert backward_call(lib, problem(**{name + "__token": 64, name + "__head": 64})) == cuvit.ERROR_INVALID_ARGUMENT
    assert b"overlap" in lib.cuvit_last_error()


LENGTH = [dict(heads=65536, kv_heads=65536, tokens=1, kv_tokens=1), dict(tokens=INT_MAX // 4 + 1),
          dict(kv_tokens=INT_MAX // 2 + 1, tokens=1), dict(q__token=2 ** 22 + 8), dict(v__token=2 ** 40),
          dict(sequences=2 ** 24, tokens=1, kv_tokens=1)]


@CALLS
@pytest.mark.parametrize("fields", LENGTH, ids=[str(f) for f in LENGTH])
def test_too_large(lib, call, fields):
    assert call(lib, problem(**fields), kv_starts=ADDRESS) == cuvit.ERROR_LENGTH


@CALLS
@pytest.mark.parametrize("name", ["q", "k", "v", "starts", "out"])
def test_null_operands(lib, call, name):
    assert call(lib, problem(), **{name: None}) == cuvit.ERROR_INVALID_ARGUMENT
    assert call(lib, None) == cuvit.ERROR_INVALID_ARGUMENT


@pytest.mark.parametrize("name", ["lse", "grad_out", "grad_q", "grad_k", "grad_v"])
def test_null_gradients(lib, name):
    assert backward_call(lib, problem(), **{name: None}) == cuvit.ERROR_INVALID_ARGUMENT


@CALLS
@pytest.mark.parametrize("bf16", [False, True])
def test_alignment(lib, call, bf16):
    for name in ("q", "k", "v", "out"):
        assert call(lib, problem(), bf16=bf16, **{name: ADDRESS * 4 + 8}) == cuvit.ERROR_INVALID_ARGUMENT
    assert call(lib, problem(), bf16=bf16, starts=ADDRESS + 2) == cuvit.ERROR_INVALID_ARGUMENT
    assert call(lib, problem(), bf16=bf16, lse=ADDRESS + 2) == cuvit.ERROR_INVALID_ARGUMENT


def test_in_place_and_workspaces(lib):
    assert forward_call(lib, problem(), out=ADDRESS) == cuvit.ERROR_INVALID_ARGUMENT
    for name in ("grad_q", "grad_k", "grad_v"):
        assert backward_call(lib, problem(), **{name: ADDRESS}) == cuvit.ERROR_INVALID_ARGUMENT
    needed = cuvit.packed_attention_backward_workspace(problem())
    assert needed > 0
    for bad in (dict(workspace=None), dict(workspace=ADDRESS + 8), dict(nbytes=needed - 1)):
        assert backward_call(lib, problem(), **bad) == cuvit.ERROR_INVALID_ARGUMENT
        assert b"workspace" in lib.cuvit_last_error()


@pytest.mark.parametrize("fields", [dict(sequences=0), dict(heads=-1), dict(head_dim=60), dict(kv_heads=3)])
def test_no_workspace_for_what_is_refused(fields):
    assert cuvit.packed_attention_workspace(problem(**fields)) == 0
    assert cuvit.packed_attention_backward_workspace(problem(**fields)) == 0


@CALLS
def test_keys_of_another_count_need_their_starts(lib, call):
    assert call(lib, problem(kv_tokens=11)) == cuvit.ERROR_INVALID_ARGUMENT
    assert b"kv_starts" in lib.cuvit_last_error()


def test_problem_fields():
    p = cuvit.packed_attention_problem(3, 50, 6, 80, kv_heads=2, causal=True, projection=True)
    assert (p.sequences, p.tokens, p.kv_tokens, p.heads, p.kv_heads, p.head_dim) == (3, 50, 50, 6, 2, 80)
    assert p.causal == 1 and p.scale == 0.0
    assert [(s.token, s.head) for s in (p.q, p.k, p.v, p.out)] == [(800, 80)] * 3 + [(0, 0)]
    cuvit.library().cuvit_packed_attention_problem_init(None, 1, 1, 1, 1)  # ignored, as the other ones
    cuvit.library().cuvit_packed_attention_problem_projection(None)


def test_python_refusals():
    x = torch.zeros(10, 4, 64)
    p = problem()
    with pytest.raises(cuvit.InvalidArgument, match="not a GPU tensor"):
        cuvit.packed_attention(x, x, x, x, x, p)
    with pytest.raises(cuvit.InvalidArgument, match="strides"):
        cuvit.packed_attention(x, None, None, x, x, p)  # packed strides, yet a projection
    with pytest.raises(cuvit.InvalidArgument, match="as many keys"):
        cuvit.packed_attention(x, None, None, x, x, problem(kv_tokens=3))
    with pytest.raises(cuvit.InvalidArgument, match="one tensor"):
        cuvit.packed_attention_backward(x, None, None, x, x, x, x, x, x, x, p)


@pytest.mark.parametrize("causal", [False, True])
def test_formula_against_differences(causal):
    """Central differences of the 64-bit forward along random directions: off by h^2 / 6
    times its third derivative (below 100 for values of about 1) and 2^-50 / h of rounding."""
    p = Packed([3, 0, 4], 4, 8, kv_heads=2, keys=[5, 2, 3], causal=causal, spare=1)
    generator = seeded(5)
    operands = [normal(generator, p.tokens, 4, 8).double()] + [normal(generator, p.kv_tokens, 2, 8).double()
                                                               for _ in range(2)]
    grad = normal(generator, p.tokens, 4, 8).double()
    exact, _ = gradients(p, *operands, grad, torch.float32)
    h = 1e-4
    for i in range(3):
        direction = normal(generator, *operands[i].shape).double()

        def value(step):
            moved = [x + step * direction if j == i else x for j, x in enumerate(operands)]
            return float((forward(p, *moved, torch.float32)[0] * grad).sum())

        difference = (value(h) - value(-h)) / (2.0 * h)
        assert abs(difference - float((exact[i] * direction).sum())) < 2e-6
