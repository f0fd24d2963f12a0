"""Every kernel of the feed-forward block's products on the GPU against the FP64 definition: tiles of all sizes, cut and
whole depths, gradients in one launch and in three, of packed operands and of those that are multiplied where they lie (sizes:
tests/feed_forward_sizes.py).  Bounds as in tests/feed_forward_reference.py."""

from __future__ import annotations

import pytest
import torch

from feed_forward_sizes import RAGGED, RAGGED_FP32, WHOLE, WHOLE_FP32
from test_gpu_feed_forward import BF16, FP16, FP32, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,activation", [(BF16, "silu"), (FP16, "gelu")])
@pytest.mark.parametrize("sizes", RAGGED)
def test_packed(sizes, dtype, activation):
    _check(*_inputs(61, *sizes, dtype), activation)


@pytest.mark.parametrize("dtype,activation", [(BF16, "gelu"), (FP16, "silu")])
@pytest.mark.parametrize("sizes", WHOLE)
def test_in_place(sizes, dtype, activation):
    _check(*_inputs(62, *sizes, dtype), activation, recompute=dtype == BF16)


@pytest.mark.parametrize("sizes", RAGGED_FP32)
def test_fp32_packed(sizes):
    _check(*_inputs(63, *sizes, FP32), "silu")


@pytest.mark.parametrize("sizes", WHOLE_FP32)
def test_fp32_in_place(sizes):
    _check(*_inputs(64, *sizes, FP32), "gelu")
