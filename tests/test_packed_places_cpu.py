"""Where packed attention's tiles and workgroups lie (kernels/packed_places.hpp): every
tile of every sequence has one workgroup, and no start or length, whatever it holds,
places a row outside the operands. The C++ launchers' refusals are here too."""

from __future__ import annotations

import ctypes
import random
import subprocess
from pathlib import Path

import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def places():
    library = Path(ROOT) / "tests" / "cpp" / "bin" / "libpacked_places.so"
    if not library.exists():
        subprocess.run(["make", "-s", "-C", str(library.parents[1])], check=True)
    loaded = ctypes.CDLL(str(library))
    loaded.packed_slots.restype = ctypes.c_int64
    loaded.packed_items.restype = ctypes.c_int64
    loaded.packed_items.argtypes = [ctypes.c_int64, ctypes.c_int]
    return loaded


def ints(values):
    return (ctypes.c_int32 * len(values))(*values)


@pytest.mark.parametrize("rows", [16, 32, 64, 128])
@pytest.mark.parametrize("times", [1, 3, 16])
def test_every_tile_has_one_slot(places, rows, times):
    rng = random.Random(rows * times)
    for _ in range(40):
        lengths = [rng.choice([0, 0, 1, rng.randint(0, 300)]) for _ in range(rng.randint(1, 150))]
        starts = [rng.randint(0, 50)]
        for n in lengths:
            starts.append(starts[-1] + n)
        tokens = starts[-1] + rng.randint(0, 40)
        table = ints(starts)
        slots = places.packed_slots(tokens, times, rows, len(lengths))
        firsts = [places.packed_first_slot(table, s, tokens, times, rows) for s in range(len(lengths))]
        assert all(a < b for a, b in zip(firsts, firsts[1:]))
        for s, n in enumerate(lengths):
            tiles = -(-n * times // rows)
            behind = firsts[s + 1] if s + 1 < len(lengths) else slots
            assert firsts[s] + tiles <= behind  # the slots firsts[s] + tile are this sequence's


@pytest.mark.parametrize("last_first", [0, 1])
@pytest.mark.parametrize("slots,heads", [(1, 1), (7, 3), (64, 12), (33, 65), (1000, 1)])
def test_every_slot_has_one_workgroup(places, slots, heads, last_first):
    out = ints([0, 0])
    seen = set()
    for block in range(places.packed_items(slots, heads) + 9):
        places.packed_item(ctypes.c_uint32(block), slots, heads, last_first, out)
        if out[0] >= 0:
            assert 0 <= out[0] < heads and 0 <= out[1] < slots
            assert (out[0], out[1]) not in seen
            seen.add((out[0], out[1]))
    assert len(seen) == slots * heads


def test_spans_stay_within_the_operands(places):
    rng = random.Random(5)
    extremes = [-2 ** 31, -1, 0, 1, 2 ** 31 - 1]
    out = ints([0] * 4)
    for _ in range(3000):
        tokens, keys = rng.choice([0, 1, 50, 2 ** 31 - 1]), rng.choice([0, 1, 70, 2 ** 31 - 1])

        def value(limit):
            return rng.choice(extremes + [rng.randint(-5, 80), rng.randint(0, limit)])

        starts = ints([value(tokens) for _ in range(3)])
        kv_starts = ints([value(keys) for _ in range(3)])
        lengths = ints([value(keys) for _ in range(2)])
        for s in range(2):
            places.packed_span(starts, kv_starts, rng.choice([None, lengths]), tokens, keys, s, out)
            assert 0 <= out[0] and 0 <= out[1] and out[0] + out[1] <= tokens
            assert 0 <= out[2] and 0 <= out[3] and out[2] + out[3] <= keys


@pytest.mark.parametrize("tokens,heads,head_dim", [(1, 1, 64), (5, 3, 80), (2 ** 31 - 1, 1, 256), (3, 65535, 256)])
def test_what_operands_reach(places, tokens, heads, head_dim):
    places.packed_reach.restype = ctypes.c_int64
    places.packed_reach.argtypes = [ctypes.c_int] * 3 + [ctypes.c_int64] * 2
    strides = [0, 1, 64, 2 ** 22, 2 ** 31, 2 ** 40, 2 ** 40 + 1, 2 ** 62, 2 ** 63 - 1, -1, -2 ** 63]
    for token in strides:
        for head in strides:
            produced = places.packed_reach(tokens, heads, head_dim, token, head)
            exact = (tokens - 1) * (token or heads * head_dim) + (heads - 1) * (head or head_dim) + head_dim
            assert produced == -1 if min(token, head) < 0 else produced in (-1, exact)
            if 0 <= min(token, head) and max(token, head) <= 64 and exact < 2 ** 31:
                assert produced == exact
    assert places.packed_reach(0, heads, head_dim, 0, 0) == -1


PROGRAM = r"""
#include <cuvit/kernels.hpp>
#include <cstdio>
#include <stdexcept>

template <typename Call> int refused(Call&& call) {
    try {
        call();
    } catch (const std::invalid_argument&) {
        return 1;
    }
    return 0;
}

int main() {
    cuvit::PackedAttentionProblem attention;
    cuvit_packed_attention_problem_init(&attention, 1, 4, 2, 60); // no multiple of 8
    cuvit::GatedProblem gated;
    cuvit_gated_problem_init(&gated, 4, 8, 8, CUVIT_GATE_SILU);
    const cuvit::PackedSequences none;
    float* const f = nullptr;
    std::uint16_t* const h = nullptr;
    std::uint8_t* const b = nullptr;
    int count = 0;
    count += refused([&] { cuvit::launch_packed_attention(f, f, f, none, f, f, attention); });
    count += refused([&] { cuvit::launch_packed_attention(h, h, h, none, h, f, attention); });
    count += refused([&] { cuvit::launch_packed_attention_backward(f, f, f, none, f, f, f, f, f, f, attention); });
    count += refused([&] { cuvit::launch_packed_attention_backward(h, h, h, none, h, f, h, h, h, h, attention); });
    count += refused([&] { cuvit::launch_gated_checkpoint_gemm(f, f, f, f, b, b, gated); });
    count += refused([&] { cuvit::launch_gated_checkpoint_gemm(h, h, f, h, b, b, gated); });
    count += refused([&] { cuvit::launch_gated_checkpoint_backward(b, b, f, f, f, gated); });
    count += refused([&] { cuvit::launch_gated_checkpoint_backward(b, b, h, h, h, gated); });
    attention.tokens = 0; // nothing to do
    cuvit::launch_packed_attention(f, f, f, none, f, f, attention);
    std::printf("%d\n", count);
}
"""


def test_launchers_refuse_as_the_c_abi(tmp_path):
    source, program = tmp_path / "launchers.cpp", tmp_path / "launchers"
    source.write_text(PROGRAM)
    lib = Path(ROOT) / "cu-vit_amd" / "lib"
    subprocess.run(["/opt/rocm/bin/hipcc", "-O0", "-std=c++17", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT}/include",
                    "-I/opt/rocm/include", "-x", "c++", str(source), "-o", str(program), f"-L{lib}", "-lcuvit_amd",
                    "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{lib}"], check=True)
    assert subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout == "8\n"
