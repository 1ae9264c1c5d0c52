"""Every tile of every product of the gated feed-forward block, whole and cut along its sum, at sizes that the rules send there.

The variants are asked for first (``qsrt_gated_ffn_plan``), so that a rule that changes does not leave one untested.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from qsrt_amd import _native
from qsrt_amd.gated_ffn import gated_ffn, gated_ffn_gradients
from test_gated_ffn_gpu import check, draw, want

pytestmark = pytest.mark.gpu
SQUARE, WIDE, SMALL, FLAT, ROWS = range(5)

# tokens, hidden, inter: the tile, and whether the sum is cut, of gate and up, down, dM, dx, the weights' gradients
CASES = {
    (1, 72, 72): ((ROWS, 0), (ROWS, 0), (FLAT, 0), (FLAT, 1), (SMALL, 0)),
    (7, 4104, 2056): ((ROWS, 0), (ROWS, 0), (FLAT, 1), (FLAT, 1), (SQUARE, 0)),  # waves' parts of 16 and 17 steps
    (16, 4096, 520): ((ROWS, 0), (ROWS, 0), (FLAT, 1), (FLAT, 1), (WIDE, 0)),  # of 16, of four and five
    (17, 72, 72): ((FLAT, 0), (FLAT, 0), (FLAT, 0), (FLAT, 1), (SMALL, 0)),
    (24, 520, 264): ((FLAT, 1), (FLAT, 1), (FLAT, 1), (FLAT, 1), (SMALL, 0)),
    (24, 520, 72): ((FLAT, 1), (FLAT, 0), (FLAT, 1), (FLAT, 1), (SMALL, 0)),
    (32, 6152, 72): ((FLAT, 1), (FLAT, 0), (FLAT, 1), (FLAT, 0), (SMALL, 0)),
    (33, 72, 264): ((SMALL, 0), (SMALL, 1), (SMALL, 0), (SMALL, 1), (SMALL, 0)),
    (33, 520, 72): ((SMALL, 1), (SMALL, 0), (SMALL, 1), (SMALL, 0), (SMALL, 0)),
    (65, 72, 72): ((SMALL, 0), (SMALL, 0), (SMALL, 0), (SMALL, 0), (SMALL, 0)),
    (33, 2568, 6152): ((WIDE, 1), (SMALL, 1), (SMALL, 1), (SMALL, 1), (SQUARE, 0)),
    (33, 5128, 8200): ((WIDE, 1), (SMALL, 1), (WIDE, 1), (WIDE, 1), (SQUARE, 0)),
    (33, 8200, 2568): ((SMALL, 1), (WIDE, 1), (SMALL, 1), (WIDE, 1), (SQUARE, 0)),
    (130, 72, 8200): ((WIDE, 0), (SMALL, 1), (SMALL, 0), (SMALL, 1), (SMALL, 0)),
    (390, 72, 8200): ((SQUARE, 0), (SMALL, 1), (WIDE, 0), (SMALL, 1), (SMALL, 0)),
    (390, 8200, 72): ((SMALL, 1), (WIDE, 0), (SMALL, 1), (WIDE, 0), (SMALL, 0)),
    (900, 72, 8200): ((SQUARE, 0), (SMALL, 1), (SQUARE, 0), (SMALL, 1), (SMALL, 0)),
    (900, 8200, 72): ((SMALL, 1), (SQUARE, 0), (SMALL, 1), (SQUARE, 0), (SMALL, 0)),
    (130, 8200, 6152): ((SQUARE, 1), (SQUARE, 1), (WIDE, 1), (SQUARE, 1), (SQUARE, 0)),
    (130, 6152, 8200): ((SQUARE, 1), (WIDE, 1), (SQUARE, 1), (SQUARE, 1), (SQUARE, 0)),
    (130, 2568, 8200): ((SQUARE, 1), (SMALL, 1), (SMALL, 0), (SMALL, 1), (SQUARE, 0)),
}


def plan_of(t, hidden, inter):
    plan = (ctypes.c_int64 * 11)()
    _native.check(_native.lib().qsrt_gated_ffn_plan(t, hidden, inter, plan), "qsrt_gated_ffn_plan")
    return tuple((plan[i], int(plan[i + 1] > 1)) for i in range(0, 10, 2)), plan[10]


def test_the_cases_take_every_variant():
    taken = [{variants[i] for variants in CASES.values()} for i in range(5)]
    tiles = {(tile, cut) for tile in (SQUARE, WIDE, SMALL, FLAT) for cut in (0, 1)}
    assert taken[0] == taken[1] == tiles | {(ROWS, 0)} and taken[2] == taken[3] == tiles
    assert taken[4] == {(tile, 0) for tile in (SQUARE, WIDE, SMALL)}


@pytest.mark.parametrize("sizes", CASES)
def test_variants(sizes):
    variants, pieces = plan_of(*sizes)
    assert pieces == (2 if sizes[0] <= 64 else 1)
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert variants == CASES[sizes]
    dtype = (torch.bfloat16, torch.float16)[sum(sizes) // 8 % 2]
    x, gate, up, down, dy = draw(sum(sizes), *sizes, dtype)
    expected = want(x, gate, up, down, dy, "swiglu", pieces)
    check({"y": gated_ffn(x, gate, up, down)}, expected, ["y"])
    check(vars(gated_ffn_gradients(x, dy, gate, up, down)), expected, ["middle", "gate_rows", "up_rows", "x", "gate", "up", "down"])
