"""How packed attention is divided (kernels/packed_choice.hpp) on the 256 compute units of
an MI355X: that the GPU tests reach every kernel, and the measured sizes theirs. Which keys
the parts and the queries take (kernels/packed_places.hpp), up to the longest caches that a
call accepts; and that none longer is."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

import cuvit_amd as cuvit
from conftest import ROOT
from packed_support import Packed
from test_packed_attention_cpu import ADDRESS, CALLS, backward_call, forward_call
from test_packed_divisions_gpu import FORWARD, GRADIENTS, HEAD_DIMS

MOST = 2 ** 31 - 1
UNITS = 256
KINDS = ["parts", "few", "middle", "large"]
WIDTHS = [32, 64, 96, 128, 256]  # that kernels are built for


def sizes(sequences, tokens, kv_tokens, heads, kv_heads, head_dim):
    return (ctypes.c_int32 * 6)(sequences, tokens, kv_tokens, heads, kv_heads, head_dim)


def width(head_dim):
    return next(w for w in WIDTHS if head_dim <= w)


def sizes_of(case, head_dim):
    queries, keys, heads, kv_heads = case
    p = Packed(queries, heads, head_dim, kv_heads=kv_heads, keys=keys)
    return sizes(len(queries), p.tokens, p.kv_tokens, heads, kv_heads, head_dim)


def forward_kind(choice, problem, single):
    parts = ctypes.c_int32()
    kind = KINDS[choice.packed_forward_choice(problem, single, UNITS, ctypes.byref(parts))]
    assert (parts.value >= 4) == (kind == "parts")
    return kind


@pytest.fixture(scope="module")
def choice():
    library = Path(ROOT) / "tests" / "cpp" / "bin" / "libpacked_choice.so"
    if not library.exists():
        subprocess.run(["make", "-s", "-C", str(library.parents[1])], check=True)
    return ctypes.CDLL(str(library))


@pytest.mark.parametrize("keys", [0, 1, 31, 32, 33, 4096, 12545, 2 ** 30 + 7, 2 ** 31 - 4096, MOST - 99, MOST - 31,
                                  MOST - 30, MOST])
@pytest.mark.parametrize("parts", [4, 7, 64, 512, 2048, 2432])
def test_parts_cover_the_keys(choice, keys, parts):
    """One behind the other, from the first key to the last, whole blocks each but the last one."""
    out = (ctypes.c_int32 * 2)()
    at = 0
    for part in range(parts):
        choice.packed_part(keys, part, parts, 32, out)
        assert out[0] == at and at <= out[1] <= keys
        assert out[0] == keys or out[0] % 32 == 0
        at = out[1]
    assert at == keys


def test_keys_that_a_query_sees(choice):
    counts = [0, 1, 2, 5000, 2 ** 30, 2 ** 31 - 4096, MOST]
    for queries in counts[1:]:
        for keys in counts:
            for query in {0, 1, queries // 2, queries - 1}:
                if query < queries:
                    expected = min(max(query + 1 + keys - queries, 0), keys)
                    assert choice.packed_seen(query, queries, keys, 1) == expected
                    assert choice.packed_seen(query, queries, keys, 0) == keys


LONGEST = 2 ** 31 - 4096


def single_head(tokens, kv_tokens):
    return cuvit.packed_attention_problem(1, tokens, 1, 8, kv_tokens=kv_tokens)


@CALLS
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("tokens,kv_tokens", [(1, LONGEST + 1), (LONGEST + 1, 1), (1, MOST), (MOST, 1), (MOST, MOST)])
def test_lengths_near_2_to_31(lib, call, bf16, tokens, kv_tokens):
    """The walks over keys and queries step past the last one in 32 bits."""
    assert call(lib, single_head(tokens, kv_tokens), bf16=bf16, kv_starts=ADDRESS) == cuvit.ERROR_LENGTH
    assert b"2^31 - 4096" in lib.cuvit_last_error()


def test_the_longest_lengths_are_taken(lib):
    """Refused only for what is checked behind the lengths."""
    for tokens, kv_tokens in ((1, LONGEST), (LONGEST, 1), (LONGEST, LONGEST)):
        assert forward_call(lib, single_head(tokens, kv_tokens), kv_starts=ADDRESS, q=ADDRESS + 8) == cuvit.ERROR_INVALID_ARGUMENT
        assert b"aligned" in lib.cuvit_last_error()


def test_gradients_are_refused_before_any_launch(lib):
    """Keys for more than 2^32 threads, queries for few: nothing is overwritten. (Without a
    GPU the rows' launch would end the call with another error.)"""
    p = cuvit.packed_attention_problem(1, 1, 1, 8, kv_tokens=2 ** 30)
    assert backward_call(lib, p, bf16=False, kv_starts=ADDRESS) == cuvit.ERROR_LENGTH
    assert b"2^32 threads" in lib.cuvit_last_error()


@pytest.mark.parametrize("single", [0, 1])
def test_the_gpu_cases_reach_every_forward(choice, single):
    reached = set()
    for name, case in FORWARD.items():
        for head_dim in HEAD_DIMS:
            kind = forward_kind(choice, sizes_of(case, head_dim), single)
            # (fp32 has no larger tiles than the pairs'.)
            assert kind == ("middle" if single and name == "large" else name.split("_")[0]), (name, head_dim)
            reached.add((kind, width(head_dim)))
    assert reached == {(kind, w) for kind in KINDS for w in WIDTHS if not single or kind != "large"}


@pytest.mark.parametrize("single", [0, 1])
def test_the_gpu_cases_reach_every_gradient(choice, single):
    rows, keys = set(), set()
    for name, case in GRADIENTS.items():
        for head_dim in HEAD_DIMS:
            problem = sizes_of(case, head_dim)
            rows.add((choice.packed_query_sharing(problem, single, UNITS), width(head_dim)))
            keys.add((choice.packed_key_sharing(problem, single, UNITS), width(head_dim)))
    every = {(n, w) for n in ((2, 4) if single else (1, 2, 4)) for w in WIDTHS if n < 4 or w <= 128}
    assert rows == every and keys == every


@pytest.mark.parametrize("sequences,tokens,kv_tokens,heads,kv_heads,head_dim,single,expected", [
    (1, 197, 197, 3, 3, 64, 1, "few"), (64, 64 * 577, 64 * 577, 12, 12, 64, 0, "large"),
    (1, 3136, 3136, 12, 12, 64, 0, "middle"), (4, 4 * 577, 4 * 577, 6, 6, 64, 0, "few"),
    (16, 16, 16 * 12545, 12, 4, 128, 0, "parts"), (64, 64, 64 * 8192, 12, 4, 128, 0, "parts"),
    (256, 256, 256 * 2048, 32, 8, 128, 0, "middle"), (1024, 1024, 1024 * 577, 12, 12, 64, 0, "middle")])
def test_measured_sizes(choice, sequences, tokens, kv_tokens, heads, kv_heads, head_dim, single, expected):
    assert forward_kind(choice, sizes(sequences, tokens, kv_tokens, heads, kv_heads, head_dim), single) == expected


@pytest.mark.parametrize("single", [0, 1])
@pytest.mark.parametrize("sequences", [2 ** 20, 2 ** 22 - 1, 2 ** 22, 5_000_000, 2 ** 23 - 1, 2 ** 24])
def test_short_walks_are_not_shared_however_many_sequences(choice, single, sequences):
    """(On more compute units than there are tiles, so that the walk alone decides.)"""
    problem = sizes(sequences, sequences, sequences, 1, 1, 64)
    for sharing in (choice.packed_query_sharing, choice.packed_key_sharing):
        assert sharing(problem, single, 2 ** 28) == (2 if single else 1)


@pytest.mark.parametrize("sequences,queries,keys,heads,kv_heads,head_dim,single,expected", [
    # Prompts, and few queries over short caches: the join would take longer than the walk.
    (4, 577, 577, 6, 6, 64, 0, "few"), (1, 577, 577, 6, 6, 64, 0, "few"), (1, 785, 785, 12, 4, 128, 0, "few"),
    (1, 577, 577, 6, 6, 64, 1, "few"), (4, 256, 2048, 6, 6, 64, 0, "few"), (1, 577, 2048, 6, 6, 64, 1, "few"),
    (1, 256, 2048, 12, 4, 128, 1, "few"), (1, 1, 577, 6, 6, 64, 0, "few"), (4, 16, 577, 12, 4, 128, 1, "few"),
    # Few rows over long ones.
    (1, 1, 2048, 6, 6, 64, 0, "parts"), (1, 64, 2048, 6, 6, 64, 0, "parts"), (4, 16, 2048, 12, 4, 128, 1, "parts"),
    (4, 64, 2048, 6, 6, 64, 1, "parts"), (1, 577, 12545, 6, 6, 64, 0, "parts"), (4, 1, 12545, 12, 4, 128, 1, "parts")])
def test_parts_where_the_join_is_the_shorter(choice, sequences, queries, keys, heads, kv_heads, head_dim, single,
                                             expected):
    problem = sizes(sequences, sequences * queries, sequences * keys, heads, kv_heads, head_dim)
    assert forward_kind(choice, problem, single) == expected


@CALLS
@pytest.mark.parametrize("bf16", [False, True])
def test_scales_that_leave_the_exponents_no_room(lib, call, bf16):
    """The exponent's base 2 takes 1.4427 times the scale, which has to be finite."""
    for scale in (1.8e38, 2.3e38, 2.4e38, 3.4028234663852886e38):
        p = cuvit.packed_attention_problem(2, 10, 4, 64, kv_heads=2, scale=scale)
        assert call(lib, p, bf16=bf16) == cuvit.ERROR_INVALID_ARGUMENT
        assert b"scale" in lib.cuvit_last_error()
        assert cuvit.packed_attention_workspace(p) == 0 and cuvit.packed_attention_backward_workspace(p) == 0


def test_the_largest_and_smallest_scales_are_taken(lib):
    for scale in (2.0 ** 127, 2.0 ** -126):
        p = cuvit.packed_attention_problem(2, 10, 4, 64, kv_heads=2, scale=scale)
        assert forward_call(lib, p, q=ADDRESS + 8) == cuvit.ERROR_INVALID_ARGUMENT
        assert b"aligned" in lib.cuvit_last_error()


@CALLS
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_strides_near_2_to_63(lib, call, bf16, name):
    """Whole pieces or not, without a product that overflows."""
    for stride, expected in ((2 ** 62, cuvit.ERROR_LENGTH), (2 ** 63 - 8, cuvit.ERROR_LENGTH),
                             (2 ** 63 - 1, cuvit.ERROR_INVALID_ARGUMENT), (2 ** 61 + 1, cuvit.ERROR_INVALID_ARGUMENT)):
        for field in ("token", "head"):
            p = cuvit.packed_attention_problem(2, 10, 4, 64, kv_heads=2)
            setattr(getattr(p, name), field, stride)
            assert call(lib, p, bf16=bf16) == expected
