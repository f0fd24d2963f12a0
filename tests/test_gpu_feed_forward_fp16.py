"""FP16 upstream gradients of the feed-forward block on the GPU: those of a mean over many tokens are far below 1, and their
projections' gradients are formed at a power of two of them, so that FP16's least numbers cost nothing.  Bounds as in
tests/feed_forward_reference.py; `_norm_bounds` derives those of small gradients."""

from __future__ import annotations

import math

import pytest
import torch

import feed_forward_reference as reference
from attnres import layers
from layer_reference import FLOOR, assert_within
from test_gpu_feed_forward import FP16, NAMES, _inputs, _run

pytestmark = pytest.mark.gpu

LEAST_NORMAL = 2.0**-14


def _norm_bounds(x, gate_up, down, grad, values, norms):
    """The relative norms of large random inputs and, of small gradients, half a step of the least numbers: of the results' own,
    and of the projections' gradients' at a power of two that takes the largest upstream gradient to 1/4 at least.  Their
    errors are independent of what they are multiplied by, so a product's is the norms' product."""
    step = FLOOR[FP16] * 4 * float(grad.abs().max())
    hidden = down.shape[1]
    of_sums = (0.0, step * math.sqrt(x.shape[0]) * float(gate_up.double().norm()), step * math.sqrt(2 * hidden) * float(x.double().norm()), 0.0)
    return [norm + (FLOOR[FP16] * math.sqrt(value.numel()) + of_sum) / float(value.norm())
            for value, norm, of_sum in zip(values, norms, of_sums)]


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("magnitude,spread", [(2e-6, 0.0), (1e-5, 0.0), (1e-5, 1.5), (1e-3, 1.5), (1.0, 0.0), (300.0, 0.0)])
@pytest.mark.parametrize("sizes", [(512, 1024, 704, 1024), (2051, 260, 300, 129)])
def test_small_upstream_gradients(sizes, magnitude, spread, activation):
    x, gate_up, down, _grad = _inputs(51, *sizes, FP16)
    x = (x.float() / 4).to(FP16)  # rows of 300 times as much gradient stay below FP16's largest
    g = torch.Generator(device="cuda").manual_seed(52)
    rows = torch.exp(spread * torch.randn(sizes[0], 1, generator=g, device="cuda"))
    grad = (magnitude * rows * torch.randn(sizes[0], sizes[3], generator=g, device="cuda")).to(FP16)
    results = _run(x, gate_up, down, grad, activation=activation)
    values, _bounds, norms = reference.feed_forward(x, gate_up, down, activation, grad)
    for name, actual, value, bound in zip(NAMES, results, values, _norm_bounds(x, gate_up, down, grad, values, norms)):
        finite = value.abs() < 65504.0
        off = float((actual.double() - value)[finite].norm() / value.norm())
        assert off <= bound, (name, off, bound)


@pytest.mark.parametrize("sizes", [(4096, 96, 64, 40), (40, 96, 64, 41), (700, 512, 640, 256)])
@pytest.mark.parametrize("power", [-8, -14])
def test_a_power_of_two_of_the_upstream_gradients_is_one_of_the_gradients(sizes, power):
    """The largest upstream gradient is taken to the same power of two in both calls.  At 2^-8 of multiples of 2^-6 every operand of a
    product is the same power of two of the other call's and a normal number in both, so the sums are too, and so are the results
    where they are normal numbers (a sum just below those may round up to the least of them, in shorter steps in the larger call: so
    by the larger call's result).  At 2^-14 the upstream gradients are no normal numbers, which the matrix instructions
    align otherwise: the sums differ in FP32's last places, and two roundings of half a step each may end a step apart."""
    x, gate_up, down, grad = _inputs(53, *sizes, FP16)
    grad = (grad.float().clamp(-1.75, 1.75) * 16).round() / 64  # multiples of 2^-6 below 1/2, and one above 1/4
    grad[0, 0] = 0.4375
    large = _run(x, gate_up, down, grad.to(FP16))
    small = _run(x, gate_up, down, (grad * 2.0**power).to(FP16))
    assert torch.equal(large[0], small[0])
    for name, a, b in zip(NAMES[1:], large[1:], small[1:]):
        expected, actual = a.double() * 2.0**power, b.double()
        normal = expected.abs() >= LEAST_NORMAL
        assert bool(normal.any()), name
        assert power != -8 or torch.equal(actual[normal], expected[normal]), name
        assert bool(((actual - expected).abs() <= 2 * FLOOR[FP16] + 2.0**-10 * expected.abs()).all()), name


@pytest.mark.parametrize("rows", [33, 300])
def test_a_nonfinite_row_stays_in_its_own(rows):
    """It is not taken for the largest upstream gradient."""
    x, gate_up, down, grad = _inputs(54, rows, 64, 96, 64, FP16)
    grad = (grad.float() * 1e-5).to(FP16)
    clean = _run(x, gate_up, down, grad)
    for bad in (float("nan"), float("inf")):
        spoilt = grad.clone()
        spoilt[rows - 1, 3] = bad
        out, dx, _dw, ddown = _run(x, gate_up, down, spoilt)
        assert torch.equal(out, clean[0]) and torch.equal(dx[:-1], clean[1][:-1]) and not bool(dx[-1].isfinite().any())
        others = torch.arange(64, device="cuda") != 3
        assert torch.equal(ddown[others], clean[3][others]) and not bool(ddown[3].isfinite().any())


@pytest.mark.parametrize("sizes", [(1, 1, 1, 1), (5, 64, 32, 9), (100, 64, 96, 64)])
@pytest.mark.parametrize("value", [0.0, 2.0**-24, -(2.0**-24)])
def test_upstream_gradients_of_zero_and_of_the_least_number(sizes, value):
    x, gate_up, down, grad = _inputs(55, *sizes, FP16)
    grad = torch.zeros_like(grad)
    grad[-1, -1] = value
    results = _run(x, gate_up, down, grad)
    values, bounds, _norms = reference.feed_forward(x, gate_up, down, "silu", grad)
    for name, actual, expected, bound in zip(NAMES, results, values, bounds):
        assert_within(name, actual.reshape(expected.shape), expected, bound)  # with the results' own rounding
        assert value != 0.0 or name == "out" or not bool(actual.any()), name


def test_asked_for_one_by_one_and_formed_again():
    x, gate_up, down, grad = _inputs(56, 300, 96, 200, 64, FP16)
    grad = (grad.float() * 1e-5).to(FP16)
    together = _run(x, gate_up, down, grad)
    for a, b in zip(together, _run(x, gate_up, down, grad, recompute=True)):
        assert torch.equal(a, b)
    for wanted in range(3):
        leaves = [t.detach().requires_grad_(k == wanted) for k, t in enumerate((x, gate_up, down))]
        (alone,) = torch.autograd.grad(layers.gated_feed_forward(*leaves), leaves[wanted], grad)
        assert torch.equal(alone, together[1 + wanted])


def test_captured_and_replayed_with_gradients_of_other_sizes():
    """The power of two is found again in every replay."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        leaves = [t.detach().clone().requires_grad_(True) for t in _inputs(57, 300, 96, 160, 64, FP16)[:3]]
        grad = torch.zeros(300, 64, device="cuda", dtype=FP16)

        def step():
            out = layers.gated_feed_forward(*leaves)
            return (out.detach(), *torch.autograd.grad(out, leaves, grad))

        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        results = step()
    for k, magnitude in enumerate((1e-6, 3.0, 1e-3, 1e-5)):
        fresh = (_inputs(58 + k, 300, 96, 160, 64, FP16)[3].float() * magnitude).to(FP16)
        expected = _run(*(t.detach() for t in leaves), fresh)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            grad.copy_(fresh)
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, expected))
