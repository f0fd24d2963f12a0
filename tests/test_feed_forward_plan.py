"""How the feed-forward block's calls are laid out (CPU; nothing launches)."""

from __future__ import annotations

import itertools

import pytest

from attnres import _native

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
