"""The largest k of a gated product, on the CPU: one more is refused."""

from __future__ import annotations

import pytest

import cuvit_amd as cuvit
from test_blocks_cpu import call_gated, gated_problem


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 20, 50, 100])
@pytest.mark.parametrize("k", [2 ** 31 - 4095, 2 ** 31 - 1024, 2 ** 31 - 1])
def test_refused(lib, kind, m, k):
    assert call_gated(lib, gated_problem(m=m, n=1, k=k), kind=kind) == cuvit.ERROR_LENGTH
    assert lib.cuvit_last_error().decode() == "Gated products take a k of at most 2^31 - 4096"
