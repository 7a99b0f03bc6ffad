"""Which tile a gated product takes (gated_choice.hpp) on the 256 compute units of
an MI355X: each tile's cases of the GPU tests, and the measured sizes."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

from conftest import ROOT
from test_gated_gpu import TILES, TILES_F32

UNITS = 256
NAMES = ["64x32 alone", "64x64", "64x64 alone", "128x64", "192x128", "256x128", "320x128"]
NAMES_F32 = ["32x16 alone", "32x32", "32x32 alone", "64x32"]


@pytest.fixture(scope="module")
def rules():
    library = Path(ROOT) / "tests" / "cpp" / "bin" / "libgated_choice.so"
    if not library.exists():
        subprocess.run(["make", "-s", "-C", str(library.parents[1])], check=True)
    return ctypes.CDLL(str(library))


def bf16(rules, m, n, k, units=UNITS):
    px = ctypes.c_int()
    return NAMES[rules.gated_bf16_choice(m, n, k, units, ctypes.byref(px))], px.value


def test_the_gpu_cases_reach_their_tiles(rules):
    assert {name for name, *_ in TILES} == set(NAMES)
    for name, m, n, k in TILES:
        assert bf16(rules, m, n, k)[0] == name, (m, n, k)
    assert {name for name, *_ in TILES_F32} == set(NAMES_F32)
    for name, m, n, k in TILES_F32:
        assert NAMES_F32[rules.gated_f32_choice(m, n, k, UNITS)] == name, (m, n, k)


@pytest.mark.parametrize("m,expected", [(197, "64x32 alone"), (394, "64x64 alone"), (788, "64x64"), (1576, "128x64"),
                                        (3152, "256x128"), (4616, "320x128"), (9232, "320x128"), (12608, "320x128")])
def test_measured_sizes(rules, m, expected):
    assert bf16(rules, m, 2048, 768)[0] == expected


def test_every_split_has_a_tile_for_each_block(rules):
    """An XCD split never has more blocks than tiles in a direction, on a whole
    card, a part of one and a single compute unit."""
    for units in (1, 32, 255, 256, 304):
        for m in (17, 65, 300, 5000, 2 ** 30 - 1):
            for n in (1, 64, 65, 700, 9000, 2 ** 27 - 1):
                for k in (8, 768, 8192):
                    name, px = bf16(rules, m, n, k, units)
                    rows, outputs = (int(x) for x in name.split()[0].split("x"))
                    if px > 0:
                        assert px <= -(-m // rows) and 8 // px <= -(-n // outputs)
                    rules.gated_f32_choice(m, n, k, units)
