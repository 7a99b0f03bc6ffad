"""How many elements the native binding lets a rotation touch (binding/reach.hpp):
the exact number, or a refusal, for any strides that fit the struct."""

from __future__ import annotations

import ctypes
import itertools
import subprocess
from pathlib import Path

import pytest

import cuvit_amd as cuvit
from conftest import ROOT

STRIDES = [0, 1, 64, 65, 2 ** 31, 2 ** 39, 2 ** 40, 2 ** 40 + 1, 2 ** 62, 2 ** 63 - 2, 2 ** 63 - 1, -1, -2 ** 63]


@pytest.fixture(scope="module")
def reach():
    library = Path(ROOT) / "tests" / "cpp" / "bin" / "libreach.so"
    if not library.exists():
        subprocess.run(["make", "-s", "-C", str(library.parents[1])], check=True)
    function = ctypes.CDLL(str(library)).rotary_input_reach
    function.restype = ctypes.c_int64
    return lambda problem: function(ctypes.byref(problem))


@pytest.mark.parametrize("images,tokens,heads,head_dim", [(1, 1, 1, 64), (2, 5, 3, 64), (2 ** 31 - 1, 2, 2, 2),
                                                          (2, 2 ** 31 - 1, 1, 512), (1, 2, 65535, 2 ** 31 - 2)])
def test_exact_or_refused(reach, images, tokens, heads, head_dim):
    problem = cuvit.rotary_problem(images, tokens, heads, head_dim, [])
    for image, token, head in itertools.product(STRIDES, repeat=3):
        problem.input.image, problem.input.token, problem.input.head = image, token, head
        produced = reach(problem)
        if min(image, token, head) < 0:
            assert produced == -1
            continue
        exact = ((images - 1) * (image or tokens * heads * head_dim) + (tokens - 1) * (token or heads * head_dim)
                 + (heads - 1) * (head or head_dim) + head_dim)
        assert produced in (-1, exact), (image, token, head)
        if max(image, token, head) <= 65 and exact <= 2 ** 31:
            assert produced == exact
