"""Sizes of the loss's workspaces (CPU; nothing launches)."""

from __future__ import annotations

import pytest

from attnres import _native
from test_layers_api import _status

BF16, FP16, FP32 = range(3)
FORWARD, BACKWARD, BACKWARD_OF_TOTAL = range(3)


@pytest.mark.parametrize("keep", [0, 1])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_backward_of_a_total_needs_no_weighed_rows(dtype, keep):
    size = _native.load().attnres_hip_loss_workspace_bytes
    rows, vocab, width = 3000, 5000, 500
    any_reduction, total = (size(rows, vocab, width, dtype, keep, p) for p in (BACKWARD, BACKWARD_OF_TOTAL))
    padded = 3072 * 512 * (2 if dtype == FP32 else 1) * 2  # a packed copy of the rows, a power each
    assert any_reduction - total == (0 if dtype == BF16 else padded + 4 * 3072)
    few = [size(16, vocab, width, dtype, keep, p) for p in (BACKWARD, BACKWARD_OF_TOTAL)]
    assert few[0] == few[1]


def test_a_workspace_of_the_other_reduction_is_refused():
    size = _native.load().attnres_hip_loss_workspace_bytes
    bytes = size(3000, 5000, 64, FP16, 0, BACKWARD_OF_TOTAL)
    for reduction in (0, 2):
        short = bytes if reduction == 0 else bytes - 1
        assert _status("loss_backward", rows=3000, vocab=5000, dtype=FP16, reduction=reduction, bytes=short) == _native.ERR_WORKSPACE
