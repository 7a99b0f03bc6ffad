"""What the rotary, QK-norm and gated launchers refuse, and in which order, on
the CPU: none of these calls reaches a kernel."""

from __future__ import annotations

import ctypes

import pytest
import torch

import blocks_support as support
import cuvit_amd as cuvit

FAKE = 0x1000   # non-null addresses that are never dereferenced
OTHER = 0x2000


def rotary_problem(**changes):
    p = cuvit.rotary_problem(2, 5, 3, 64, [16, 16])
    return change(p, changes)


def qk_problem(**changes):
    return change(cuvit.qk_norm_problem(2, 5, 3, 64, [16, 16]), changes)


def gated_problem(**changes):
    return change(cuvit.gated_problem(4, 6, 8), changes)


def change(p, changes):
    for name, value in changes.items():
        at = p
        *path, last = name.split("__")
        for part in path:
            at = getattr(at, part)
        if last == "pairs":
            value = (ctypes.c_int * 3)(*value)
        setattr(at, last, value)
    return p


def call_rotary(lib, p, x=FAKE, positions=FAKE, frequencies=FAKE, out=OTHER, kind="f32"):
    return getattr(lib, f"cuvit_rotary_{kind}")(x, positions, frequencies, out, ctypes.byref(p) if p else None, None)


def call_qk(lib, p, x=FAKE, positions=FAKE, frequencies=FAKE, out=OTHER, kind="f32"):
    return getattr(lib, f"cuvit_qk_norm_rotary_{kind}")(x, None, None, None, None, positions, frequencies, out,
                                                        ctypes.byref(p) if p else None, None)


def call_backward(lib, p, x=FAKE, grad=FAKE, out=OTHER, gammas=(FAKE, None, None, None), workspace=FAKE, nbytes=1 << 30,
                  kind="f32"):
    return getattr(lib, f"cuvit_qk_norm_rotary_backward_{kind}")(x, None, None, FAKE, FAKE, grad, out, *gammas,
                                                                 workspace, nbytes, ctypes.byref(p) if p else None,
                                                                 None)


def call_gated(lib, p, a=FAKE, b=FAKE, c=OTHER, kind="f32"):
    return getattr(lib, f"cuvit_gated_gemm_{kind}")(a, b, None, c, None, ctypes.byref(p) if p else None, None)


def call_gated_backward(lib, p, pre=FAKE, grad=0x3000, out=OTHER, kind="f32"):
    return getattr(lib, f"cuvit_gated_backward_{kind}")(pre, grad, out, ctypes.byref(p) if p else None, None)


def test_problems_are_filled_as_the_header_says():
    p = cuvit.rotary_problem(1, 2, 3, 64, [8, 12, 12], cuvit.ROTARY_ADJACENT)
    assert (p.images, p.tokens, p.heads, p.head_dim, p.inverse) == (1, 2, 3, 64, 0)
    assert (p.rotation.pairing, p.rotation.axes, list(p.rotation.pairs), p.rotation.position_stride) == (1, 3, [8, 12, 12], 0)
    assert (p.input.image, p.input.token, p.input.head, p.output.image) == (0, 0, 0, 0)
    q = cuvit.qk_norm_problem(1, 2, 12, 80, [20, 20], norm=cuvit.NORM_LAYER, epsilon=1e-5, kv_heads=4)
    assert (q.heads, q.kv_heads, q.norm, q.rotation.axes) == (12, 4, cuvit.NORM_LAYER, 2)
    assert q.epsilon == ctypes.c_float(1e-5).value
    q = cuvit.qk_norm_problem(1, 2, 12, 80)
    assert (q.kv_heads, q.rotation.axes) == (12, 0) and q.epsilon == ctypes.c_float(1e-6).value
    g = cuvit.gated_problem(3, 4, 5, cuvit.GATE_GELU_TANH)
    assert (g.m, g.n, g.k, g.activation, g.lda, g.ldb, g.ldc, g.ld_preactivations) == (3, 4, 5, 2, 0, 0, 0, 0)
    assert (ctypes.sizeof(cuvit.RotaryProblem), ctypes.sizeof(cuvit.QkNormProblem),
            ctypes.sizeof(cuvit.GatedProblem)) == (104, 64, 32)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_zero_extents_return_first(lib, kind):
    for name in ("images", "tokens", "heads", "head_dim"):
        assert call_rotary(lib, rotary_problem(**{name: 0, "rotation__axes": 9}), None, None, None, None, kind) == 0
        assert call_qk(lib, qk_problem(**{name: 0, "norm": 7}), None, None, None, None, kind) == 0
        assert call_backward(lib, qk_problem(**{name: 0}), None, None, None, (None,) * 4, None, 0, kind) == 0
    for name in ("m", "n"):
        assert call_gated(lib, gated_problem(**{name: 0, "activation": 9}), None, None, None, kind) == 0
        assert call_gated_backward(lib, gated_problem(**{name: 0}), None, None, None, kind) == 0


MESSAGES = [
    (lambda l: call_rotary(l, None), 1, "Rotary problem cannot be null"),
    (lambda l: call_rotary(l, rotary_problem(tokens=-1)), 1, "Rotary extents cannot be negative"),
    (lambda l: call_rotary(l, rotary_problem(tokens=-1), None), 1, "Rotary extents cannot be negative"),
    (lambda l: call_rotary(l, rotary_problem(), None), 1, "Rotary operands cannot be null"),
    (lambda l: call_rotary(l, rotary_problem(), out=None), 1, "Rotary operands cannot be null"),
    (lambda l: call_rotary(l, rotary_problem(), positions=None), 1, "A rotation needs positions and frequencies"),
    (lambda l: call_rotary(l, rotary_problem(), frequencies=None), 1, "A rotation needs positions and frequencies"),
    (lambda l: call_rotary(l, rotary_problem(rotation__pairing=2)), 1, "Rotary pairing is not a cuvit_rotary_pairing value"),
    (lambda l: call_rotary(l, rotary_problem(rotation__axes=4)), 1, "A rotation takes at most three axes"),
    (lambda l: call_rotary(l, rotary_problem(rotation__axes=-1)), 1, "A rotation takes at most three axes"),
    (lambda l: call_rotary(l, rotary_problem(rotation__pairs=[-1, 3, 0])), 1, "An axis cannot have negative pairs"),
    (lambda l: call_rotary(l, rotary_problem(rotation__pairs=[16, 17, 0])), 1, "A rotation's pairs exceed the head"),
    (lambda l: call_rotary(l, rotary_problem(rotation__pairs=[2 ** 31 - 1, 2 ** 31 - 1, 0])), 1,
     "A rotation's pairs exceed the head"),
    (lambda l: call_rotary(l, rotary_problem(rotation__position_stride=-1)), 1, "The position stride cannot be negative"),
    (lambda l: call_rotary(l, rotary_problem(output__token=-64)), 1, "Rotary strides cannot be negative"),
    (lambda l: call_rotary(l, rotary_problem(head_dim=65, rotation__axes=0)), 1,
     "Rotary heads need an even head_dim of at most 512"),
    (lambda l: call_rotary(l, rotary_problem(head_dim=514)), 1, "Rotary heads need an even head_dim of at most 512"),
    (lambda l: call_rotary(l, rotary_problem(heads=65536)), 2, "Rotary launches take at most 65535 heads"),
    (lambda l: call_rotary(l, rotary_problem(images=65536, tokens=32768)), 2,
     "Rotary launches take at most 2^31 - 1 tokens"),
    (lambda l: call_rotary(l, rotary_problem(output__token=63)), 1, "Rotary output heads overlap"),
    (lambda l: call_rotary(l, rotary_problem(output__head=640, output__token=64, output__image=640)), 1,
     "Rotary output heads overlap"),
    (lambda l: call_rotary(l, rotary_problem(output__token=2 ** 62)), 1, "Rotary output heads overlap"),
    (lambda l: call_rotary(l, rotary_problem(input__token=256), out=FAKE), 1, "Rotary in place needs equal strides"),
    (lambda l: call_qk(l, None), 1, "QK norm problem cannot be null"),
    (lambda l: call_qk(l, qk_problem(heads=-3)), 1, "QK norm extents cannot be negative"),
    (lambda l: call_qk(l, qk_problem(), None), 1, "QK norm operands cannot be null"),
    (lambda l: call_qk(l, qk_problem(kv_heads=0)), 1, "QK norm needs key heads"),
    (lambda l: call_qk(l, qk_problem(norm=2)), 1, "QK norm is not a cuvit_norm value"),
    (lambda l: call_qk(l, qk_problem(epsilon=0.0)), 1, "QK norm needs a positive normal epsilon"),
    (lambda l: call_qk(l, qk_problem(epsilon=1e-40)), 1, "QK norm needs a positive normal epsilon"),
    (lambda l: call_qk(l, qk_problem(epsilon=float("nan"))), 1, "QK norm needs a positive normal epsilon"),
    (lambda l: call_qk(l, qk_problem(epsilon=float("inf"))), 1, "QK norm needs a positive normal epsilon"),
    (lambda l: call_qk(l, qk_problem(), positions=None), 1, "A rotation needs positions and frequencies"),
    (lambda l: call_qk(l, qk_problem(heads=65530, kv_heads=65530)), 2, "Rotary launches take at most 65535 heads"),
    (lambda l: call_qk(l, qk_problem(kv_heads=2 ** 31 - 1)), 2, "Rotary launches take at most 65535 heads"),
    (lambda l: call_backward(l, None), 1, "QK norm problem cannot be null"),
    (lambda l: call_backward(l, qk_problem(), grad=None), 1, "QK norm operands cannot be null"),
    (lambda l: call_backward(l, qk_problem(), out=None), 1, "QK norm operands cannot be null"),
    (lambda l: call_backward(l, qk_problem(), out=FAKE, grad=OTHER), 1,
     "QK norm gradients cannot replace the forward's input"),
    (lambda l: call_backward(l, qk_problem(), workspace=None), 1, "QK norm gradients need a 16-byte aligned workspace"),
    (lambda l: call_backward(l, qk_problem(), workspace=FAKE + 8), 1,
     "QK norm gradients need a 16-byte aligned workspace"),
    (lambda l: call_backward(l, qk_problem(), nbytes=l.cuvit_qk_norm_rotary_workspace(ctypes.byref(qk_problem())) - 1), 1,
     "QK norm gradients need a 16-byte aligned workspace"),
    (lambda l: call_gated(l, None), 1, "Gated problem cannot be null"),
    (lambda l: call_gated(l, gated_problem(m=-1)), 1, "Gated dimensions cannot be negative"),
    (lambda l: call_gated(l, gated_problem(k=-1)), 1, "Gated dimensions cannot be negative"),
    (lambda l: call_gated(l, gated_problem(), None), 1, "Gated operands cannot be null"),
    (lambda l: call_gated(l, gated_problem(activation=3)), 1, "Gated activation is not a cuvit_gate value"),
    (lambda l: call_gated(l, gated_problem(activation=-1)), 1, "Gated activation is not a cuvit_gate value"),
    (lambda l: call_gated(l, gated_problem(lda=7)), 1, "A gated leading dimension is smaller than its row"),
    (lambda l: call_gated(l, gated_problem(ldb=7)), 1, "A gated leading dimension is smaller than its row"),
    (lambda l: call_gated(l, gated_problem(ldc=5)), 1, "A gated leading dimension is smaller than its row"),
    (lambda l: call_gated(l, gated_problem(ld_preactivations=11)), 1,
     "A gated leading dimension is smaller than its row"),
    (lambda l: call_gated(l, gated_problem(n=2 ** 30)), 2, "Gated products take at most 2^30 - 1 rows and columns"),
    (lambda l: call_gated(l, gated_problem(m=2 ** 30)), 2, "Gated products take at most 2^30 - 1 rows and columns"),
    (lambda l: call_gated(l, gated_problem(m=1, n=2 ** 29, k=7)), 2, "Gated products take less than 2^32 threads"),
    (lambda l: call_gated(l, gated_problem(m=50, n=2 ** 27, k=7)), 2, "Gated products take less than 2^32 threads"),
    (lambda l: call_gated_backward(l, None), 1, "Gated problem cannot be null"),
    (lambda l: call_gated_backward(l, gated_problem(), grad=None), 1, "Gated operands cannot be null"),
    (lambda l: call_gated_backward(l, gated_problem(), out=0x3000), 1,
     "Gated gradients cannot replace the product's gradient"),
    (lambda l: call_gated_backward(l, gated_problem(ld_preactivations=11)), 1,
     "A gated leading dimension is smaller than its row"),
]


@pytest.mark.parametrize("index", range(len(MESSAGES)))
def test_refusals(lib, index):
    call, status, message = MESSAGES[index]
    assert call(lib) == status
    assert lib.cuvit_last_error().decode().startswith(message)


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros(2, 5, 3, 64)
    at, turns = torch.zeros(5, 2), torch.zeros(32)
    with pytest.raises(cuvit.InvalidArgument):
        cuvit.rotary(x, at, turns, x, rotary_problem())
    qkv = torch.zeros(2, 5, 9, 64)
    with pytest.raises(cuvit.InvalidArgument):
        cuvit.qk_norm_rotary(qkv, None, None, at, turns, qkv, qk_problem())
    with pytest.raises(cuvit.InvalidArgument):
        cuvit.qk_norm_rotary_backward(qkv, None, None, at, turns, qkv, qkv.clone(), qk_problem())
    with pytest.raises(cuvit.InvalidArgument):
        cuvit.gated_gemm(torch.zeros(4, 8), torch.zeros(12, 8), None, torch.zeros(4, 6), gated_problem())
    with pytest.raises(cuvit.InvalidArgument):
        cuvit.gated_backward(torch.zeros(4, 12), torch.zeros(4, 6), torch.zeros(4, 12), gated_problem())


def test_the_gradient_formulas_against_differences():
    """The 64-bit formulas that the kernels are held to, against central
    differences of the forward definitions: with a step of 1e-5 both the cut
    (step^2) and the rounding (1e-16 / step) stay below 1e-8 of the values."""
    g = support.seeded(5)
    heads, kv_heads, head_dim = 3, 2, 12
    qkv = support.normal(g, 2, 3, heads + 2 * kv_heads, head_dim).double()
    grad = support.normal(g, 2, 3, heads + 2 * kv_heads, head_dim).double()
    gamma = [support.normal(g, head_dim, mean=1.0).double() for _ in range(2)]
    beta = [support.normal(g, head_dim).double() for _ in range(2)]
    at = support.normal(g, 3, 2, scale=5.0)
    for layer in (False, True):
        for adjacent in (False, True):
            turn = (at, torch.tensor([1.0, 0.1, 1.0]), [2, 1], adjacent)
            out, _, d_gamma, _, d_beta, _ = support.qk_norm_gradients(qkv, grad, heads, kv_heads, layer, 1e-3, gamma, turn)

            def loss(x, gm, bt):
                return float((support.qk_norm(x, heads, kv_heads, layer, 1e-3, gm, bt, turn)[0] * grad).sum())

            step = 1e-5
            way = support.normal(g, *qkv.shape).double()
            difference = (loss(qkv + step * way, gamma, beta) - loss(qkv - step * way, gamma, beta)) / (2 * step)
            assert abs(float((out * way).sum()) - difference) < 1e-6
            way = [support.normal(g, head_dim).double() for _ in range(2)]
            moved = [[gm + s * step * w for gm, w in zip(gamma, way)] for s in (1, -1)]
            difference = (loss(qkv, moved[0], beta) - loss(qkv, moved[1], beta)) / (2 * step)
            assert abs(float((d_gamma * torch.stack(way)).sum()) - difference) < 1e-6
            moved = [[bt + s * step * w for bt, w in zip(beta, way)] for s in (1, -1)]
            difference = (loss(qkv, gamma, moved[0]) - loss(qkv, gamma, moved[1])) / (2 * step)
            assert abs(float((d_beta * torch.stack(way)).sum()) - difference) < 1e-6
    z, d = support.normal(g, 5, 14).double(), support.normal(g, 5, 7).double()
    way = support.normal(g, 5, 14).double()
    for kind in range(3):
        def product(x):
            return float((support.activation(kind, x[:, :7]) * x[:, 7:] * d).sum())

        difference = (product(z + 1e-5 * way) - product(z - 1e-5 * way)) / 2e-5
        assert abs(float((support.gated_gradient(z, d, kind, torch.float32)[0] * way).sum()) - difference) < 1e-6
