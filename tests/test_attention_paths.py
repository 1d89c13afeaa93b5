"""Which launches a case of attention makes, asked of the library, so that a rule that moves cannot empty a test without a word; and the launches in
combination against the formulas."""

import pytest

from tests.test_attention import BF, F32, test_attention_matches_the_formula_in_both_directions as matches_the_formula
from torchllmtuner_amd import _lib

CODE = {F32: 0, BF: 1}


def paths(lengths, behind, H, G, D, dtype):
    """(forward and backward sorted: 1 and 2, shares of a tile's keys in the forward, for dq, of its queries for dk and dv, parts of a group of heads)"""
    x = _lib.load().mi355_varlen_attention_paths(sum(lengths) + behind, H, G, D, len(lengths), CODE[dtype])
    return x & 3, 1 << (x >> 4 & 3), 1 << (x >> 8 & 3), 1 << (x >> 12 & 3), x >> 16


COMBINED = [
    # (lengths, rows behind, heads, key heads, head size, dtype, paths)
    (([2000, 2200], 0, 8, 2, 64, BF), (3, 2, 2, 2, 4)),        # sorted and dealt in every pass
    (([1500, 2700], 3, 8, 2, 75, BF), (3, 2, 2, 2, 4)),
    (([2100, 2100], 0, 10, 5, 128, BF), (3, 1, 2, 2, 2)),      # ... in the backward alone
    (([1500, 1300], 7, 24, 12, 64, BF), (3, 1, 1, 1, 2)),      # sorted, not dealt
    (([1100, 1200], 0, 8, 8, 64, F32), (3, 1, 1, 1, 1)),
    (([700, 1100, 1000], 0, 24, 24, 128, BF), (2, 1, 1, 1, 1)),
    (([600, 520], 7, 8, 8, 64, F32), (2, 2, 2, 2, 1)),
    (([900, 0, 1100], 0, 16, 4, 40, F32), (2, 1, 1, 1, 4)),
    (([100] * 12, 0, 8, 2, 64, BF), (0, 1, 1, 1, 4)),         # neither
]


@pytest.mark.gpu
@pytest.mark.parametrize("case,expected", COMBINED)
def test_sorted_and_dealt_tiles_match_the_formula(case, expected):
    assert paths(*case) == expected
    matches_the_formula(*case)


@pytest.mark.parametrize("case,expected", COMBINED)
def test_what_the_cases_above_reach(case, expected):
    assert paths(*case) == expected


@pytest.mark.parametrize("lengths,behind,H,G,D,bf16,fp32", [
    # (the cases of tests/test_attention.py that are there for sorted tiles and dealt keys)
    ([600, 520], 7, 8, 8, 64, (0, 1, 1, 1, 1), (2, 2, 2, 2, 1)),
    ([512, 3, 1100], 0, 16, 4, 40, (0, 1, 1, 1, 4), (2, 1, 1, 1, 4)),
    ([520], 0, 2, 1, 64, (0, 8, 8, 8, 2), (0, 8, 8, 8, 2)),
    ([1030], 5, 1, 1, 128, (0, 8, 8, 8, 1), (0, 8, 8, 8, 1)),
    ([2100], 0, 1, 1, 40, (0, 8, 8, 8, 1), (0, 4, 4, 4, 1)),
    ([2048], 0, 2, 2, 33, (0, 8, 8, 8, 1), (0, 4, 4, 4, 1)),
    ([1, 2200], 0, 4, 2, 64, (0, 4, 4, 4, 2), (3, 2, 2, 2, 2)),
    ([1500, 0, 1700, 40], 3, 1, 1, 96, (0, 4, 4, 4, 1), (0, 4, 4, 4, 1)),
    ([2300], 0, 3, 1, 200, (0, 4, 8, 4, 3), (0, 4, 4, 4, 3)),
    ([2, 1040], 0, 1, 1, 75, (0, 8, 8, 8, 1), (0, 8, 8, 8, 1)),
    ([1100, 960], 2, 8, 2, 64, (0, 1, 2, 2, 4), (3, 1, 1, 1, 4)),
    ([3000, 1100], 0, 10, 2, 128, (3, 1, 2, 2, 5), (3, 1, 1, 1, 5)),
])
def test_what_the_plain_cases_reach(lengths, behind, H, G, D, bf16, fp32):
    assert paths(lengths, behind, H, G, D, BF) == bf16
    assert paths(lengths, behind, H, G, D, F32) == fp32


def test_workspaces_hold_what_the_paths_need():
    lib = _lib.load()
    for T, H, G, D, n, dtype in [(4200, 8, 2, 64, 2, 1), (4200, 8, 2, 64, 1, 1), (1030, 1, 1, 128, 1, 0), (8192, 32, 4, 128, 4, 1), (64, 1, 1, 64, 1, 1)]:
        x = lib.mi355_varlen_attention_paths(T, H, G, D, n, dtype)
        forward = 4 * T * H * (D + 1) << (x >> 4 & 3) if x >> 4 & 3 else 0
        assert lib.mi355_varlen_attention_fwd_workspace_bytes(T, H, G, D, n, dtype) >= forward
        dq, parts = 4 * T * H * D << (x >> 8 & 3) if x >> 8 & 3 else 0, (x >> 16) << (x >> 12 & 3)
        assert lib.mi355_varlen_attention_bwd_workspace_bytes(T, H, G, D, dtype) >= 8 * T * H + dq + (8 * T * G * D * parts if parts > 1 else 0)
    for sizes in [(0, 1, 1, 64, 1, 1), (10, 3, 2, 64, 1, 1), (10, 2, 2, 257, 1, 1), (10, 2, 2, 64, 1, 2)]:
        assert lib.mi355_varlen_attention_paths(*sizes) == 0
