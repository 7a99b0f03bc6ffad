"""The large products of test_block_paths_gpu.py take tiles of 128 outputs,
whose C goes past the caches."""

from __future__ import annotations

from test_gated_choice_cpu import bf16, rules  # noqa: F401 (a fixture)


def test_the_large_products_take_wide_tiles(rules):  # noqa: F811
    for m, n, k in ((12608, 2048, 200), (12608, 1363, 72), (9232, 2048, 200), (9999, 1681, 64)):
        assert bf16(rules, m, n, k)[0] in ("192x128", "256x128", "320x128"), (m, n, k)
