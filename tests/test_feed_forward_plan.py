"""How the feed-forward block's calls are laid out (CPU; nothing launches)."""

from __future__ import annotations

import itertools

import pytest

from attnres import _native
from feed_forward_sizes import RAGGED, RAGGED_FP32, WHOLE, WHOLE_FP32

GATE_TILE, SLOPE_TILE, PRODUCT_TILE, PRODUCT_LAUNCHES, PRODUCT_PARTS, OPERAND_PARTS, THREADS = range(7)
FORWARD, BACKWARD, BACKWARD_AGAIN = range(3)
BF16, FP16, FP32 = range(3)


def plan(sizes, dtype, backward, entry):
    return _native.load().attnres_hip_gated_ffn_plan(*sizes, dtype, backward, entry)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_launches_stay_below_2_to_the_32_threads(dtype):
    """Up to the envelope's corners, ragged (packed) or not."""
    for rows, width, hidden, out_width in itertools.product(
            (1, 300, 2**20 + 1, 2**22 + 1, 2**23 + 1, 2**24), (1, 1033, 2048, 8191, 8192), (1, 32, 8192, 65535, 65536), (1, 1033, 8192)):
        if -(-rows // 256) * -(-hidden // 128) > 2**22:
            continue
        for backward in (FORWARD, BACKWARD, BACKWARD_AGAIN):
            sizes = (rows, width, hidden, out_width)
            threads = plan(sizes, dtype, backward, THREADS)
            assert 0 <= threads < 2**32, (sizes, backward, threads)


def _kernels(sizes, dtype):
    """(product, 16-bit numbers of an operand's element or 0, tile, cut into parts, launches) of a call's forward and backward."""
    operand = plan(sizes, dtype, FORWARD, OPERAND_PARTS)
    return {("gate", operand, plan(sizes, dtype, FORWARD, GATE_TILE)), ("slope", operand, plan(sizes, dtype, BACKWARD, SLOPE_TILE)),
            ("out", operand, plan(sizes, dtype, FORWARD, PRODUCT_TILE), plan(sizes, dtype, FORWARD, PRODUCT_PARTS) > 1),
            ("gradients", operand, plan(sizes, dtype, BACKWARD, PRODUCT_TILE), plan(sizes, dtype, BACKWARD, PRODUCT_PARTS) > 1),
            ("launches", operand, plan(sizes, dtype, BACKWARD, PRODUCT_LAUNCHES))}


@pytest.mark.parametrize("sizes,dtype", [(RAGGED, BF16), (RAGGED, FP16), (WHOLE, BF16), (WHOLE, FP16), (RAGGED_FP32 + WHOLE_FP32, FP32)])
def test_sizes_of_the_gpu_tests_launch_every_kernel(sizes, dtype):
    """A change of the rates that choose tiles has to bring new sizes with it.  (FP32 in three parts, of more than 2^31 rows times
    widths, leaves no gradients few enough for tiles of 64 that four sharers take.)"""
    reached = set().union(*(_kernels(s, dtype) for s in sizes))
    for operand in (1,) if dtype != FP32 else (0, 3):
        for tile in (64, 65, 66, 128, 256) if operand else (64, 65, 66, 128):
            assert {("gate", operand, tile), ("slope", operand, tile)} <= reached, tile
            for cut in (False, True):
                assert ("out", operand, tile, cut) in reached, (tile, cut)
                assert ("gradients", operand, tile, cut) in reached or (operand, tile) == (3, 66), (tile, cut)
        assert {("launches", operand, n) for n in ((1, 3) if operand else (1,))} <= reached


@pytest.mark.parametrize("sizes,dtype,backward,entry", [
    ((0, 8, 8, 8), BF16, FORWARD, THREADS), ((4, 8193, 8, 8), BF16, FORWARD, THREADS), ((4, 8, 8, 0), BF16, FORWARD, THREADS),
    ((2**24 + 1, 8, 8, 8), BF16, FORWARD, THREADS), ((4, 8, 8, 8), 3, FORWARD, THREADS), ((4, 8, 8, 8), BF16, 3, THREADS),
    ((4, 8, 8, 8), BF16, -1, THREADS), ((4, 8, 8, 8), BF16, FORWARD, THREADS + 1), ((4, 8, 8, 8), BF16, FORWARD, -1)])
def test_plans_outside_the_envelope(sizes, dtype, backward, entry):
    assert plan(sizes, dtype, backward, entry) == -1


def test_plans_of_few_rows():
    """By kernels that take no tiles, forwards alone."""
    sizes = (1, 1024, 2816, 1024)
    assert [plan(sizes, BF16, FORWARD, e) for e in range(OPERAND_PARTS)] == [0] * 5
    assert plan(sizes, BF16, BACKWARD, GATE_TILE) == 0 and plan(sizes, BF16, BACKWARD, SLOPE_TILE) > 0
    assert plan(sizes, BF16, BACKWARD, PRODUCT_LAUNCHES) == 1 and plan(sizes, FP32, FORWARD, OPERAND_PARTS) == 0
