"""The feed-forward block (attnres.layers) at the largest numbers of rows: launches of more rows than workgroups.  Rows are one
row, or a few in front of zeros, so that what they give is known from a small call; bounds as in
tests/feed_forward_reference.py."""

from __future__ import annotations

import pytest
import torch

import feed_forward_reference as reference
from attnres import layers
from layer_reference import assert_within
from test_gpu_feed_forward import BF16, _inputs, _run

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def test_the_most_rows_of_an_odd_width():
    """2^24 rows of 1033, which are packed: 35 GB."""
    x, gate_up, down, grad = _inputs(41, 1, 1033, 32, 32, BF16)
    values, bounds, _norms = reference.feed_forward(x, gate_up, down, "silu", grad)
    with torch.no_grad():
        out = layers.gated_feed_forward(x.expand(2**24, 1033), gate_up, down)
    assert_within("out", out[:1], values[0], bounds[0])
    assert bool((out == out[:1]).all())


def test_gradients_of_many_rows_of_odd_widths():
    """2^23 + 33 rows of which the rows and their gradients are packed in one launch; rows from 48 on have gradients of zero."""
    rows, few = 2**23 + 33, 48
    x, gate_up, down, grad = _inputs(42, few, 1033, 32, 1033, BF16)
    values, bounds, _norms = reference.feed_forward(x, gate_up, down, "gelu", grad)
    many_x, many_grad = x.new_zeros(rows, 1033), x.new_zeros(rows, 1033)
    many_x[:few], many_x[few:] = x, x[0]
    many_grad[:few] = grad
    results = _run(many_x, gate_up, down, many_grad, activation="gelu")
    for name, actual, value, bound in zip(("out", "dx", "dgate_up", "ddown"), results, values, bounds):
        assert_within(name, actual[:few] if name in ("out", "dx") else actual, value, bound)
    assert bool((results[0][few:] == results[0][few]).all())
    assert not bool(results[1][few:].any())
