"""What the gated product that keeps codes, and the gradient from them, refuse."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cuvit_amd as cuvit

A, B, C, D, E, F = (0x1000 * i for i in range(1, 7))  # never dereferenced


def problem(**changes):
    p = cuvit.gated_problem(4, 70, 8)
    for name, value in changes.items():
        setattr(p, name, value)
    return p


def keep(lib, p, kind, a=A, b=B, c=C, codes=D, scales=E):
    return getattr(lib, f"cuvit_gated_checkpoint_gemm_{kind}")(a, b, None, c, codes, scales,
                                                               ctypes.byref(p) if p else None, None)


def restore(lib, p, kind, codes=A, scales=B, grad=C, grad_pre=D, hidden=None):
    return getattr(lib, f"cuvit_gated_checkpoint_backward_{kind}")(codes, scales, grad, grad_pre, hidden,
                                                                   ctypes.byref(p) if p else None, None)


KINDS = pytest.mark.parametrize("kind", ["f32", "bf16"])
INT_MAX = 2 ** 31 - 1


@KINDS
def test_nothing_to_do(lib, kind):
    nothing = dict(codes=None, scales=None)
    for name in ("m", "n"):
        p = problem(**{name: 0, "activation": 9})
        assert keep(lib, p, kind, a=None, b=None, c=None, **nothing) == cuvit.OK
        assert restore(lib, p, kind, grad=None, grad_pre=None, **nothing) == cuvit.OK


@KINDS
def test_refusals(lib, kind):
    invalid, length = cuvit.ERROR_INVALID_ARGUMENT, cuvit.ERROR_LENGTH
    assert keep(lib, None, kind) == invalid and restore(lib, None, kind) == invalid
    for name in ("a", "b", "c", "codes", "scales"):
        assert keep(lib, problem(), kind, **{name: None}) == invalid
        assert b"null" in lib.cuvit_last_error()
    for name in ("codes", "scales", "grad", "grad_pre"):
        assert restore(lib, problem(), kind, **{name: None}) == invalid
        assert b"null" in lib.cuvit_last_error()
    for changes, status in ((dict(m=-1), invalid), (dict(n=-1), invalid), (dict(activation=3), invalid),
                            (dict(activation=-1), invalid), (dict(ldc=69), invalid),
                            (dict(ld_preactivations=139), invalid), (dict(m=2 ** 30), length),
                            (dict(n=2 ** 30), length)):
        assert keep(lib, problem(**changes), kind) == status
        assert restore(lib, problem(**changes), kind) == status
    for changes, status in ((dict(k=-1), invalid), (dict(lda=7), invalid), (dict(ldb=7), invalid),
                            (dict(k=INT_MAX - 4094), length), (dict(m=2 ** 29, n=2 ** 29), length)):
        assert keep(lib, problem(**changes), kind) == status
    assert restore(lib, problem(), kind, grad_pre=C) == invalid
    assert restore(lib, problem(), kind, hidden=D) == invalid


@pytest.mark.parametrize("m,n,scales", [(4, 70, 24), (1, 1, 2), (3, 32, 6), (3, 33, 12), (0, 5, 0), (-1, 5, 0),
                                        (2 ** 30 - 1, 2 ** 30 - 1, 2 * (2 ** 30 - 1) * 2 ** 25)])
def test_scales(m, n, scales):
    assert cuvit.gated_checkpoint_scales(cuvit.gated_problem(m, n, 8)) == scales


def test_python_refusals():
    x = torch.zeros(4, 140)
    with pytest.raises(cuvit.InvalidArgument, match="not a GPU tensor"):
        cuvit.gated_checkpoint_gemm(x, x, None, x, x, x, problem())
    with pytest.raises(cuvit.InvalidArgument, match="not a GPU tensor"):
        cuvit.gated_checkpoint_backward(x, x, x, x, problem())
