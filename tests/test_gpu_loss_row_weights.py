"""The loss's gradients where the upstream gradients of the rows are far apart (token weights): every row of dH is as
accurate as if it were alone."""

from __future__ import annotations

import pytest
import torch

import layer_reference as reference
from attnres import layers
from layer_reference import assert_within

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(seed, rows, width, vocab, dtype, ignored=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hidden = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    weight = (torch.randn(vocab, width, generator=g, device="cuda") * (2.0 / width**0.5)).to(dtype)
    targets = torch.randint(vocab, (rows,), generator=g, device="cuda")
    targets[torch.rand(rows, generator=g, device="cuda") < ignored] = -100
    return g, hidden, weight, targets


def _weighted(hidden, weight, targets, upstream, recompute):
    leaves = (hidden.detach().requires_grad_(True), weight.detach().requires_grad_(True))
    out = layers.linear_cross_entropy(*leaves, targets, reduction="none", recompute=recompute)
    return torch.autograd.grad(out, leaves, upstream)


@pytest.mark.parametrize("rows,width,vocab,ignored", [(64, 96, 900, 0.0), (65, 96, 900, 0.0), (300, 200, 4096, 0.0), (700, 128, 513, 0.3)])
@pytest.mark.parametrize("dtype,lowest,highest", [(BF16, -12, 0), (BF16, -9, 12), (BF16, 0, 0), (FP16, -4, 3), (FP16, 0, 0),
                                                  (FP32, -12, 0), (FP32, -9, 12), (FP32, 28, 36), (FP32, -30, -24), (FP32, 0, 0)])
@pytest.mark.parametrize("recompute", [False, True])
def test_rows_of_small_weight(rows, width, vocab, ignored, dtype, lowest, highest, recompute):
    """Weights from 10^lowest to 10^highest (what FP16 results hold).  A row's dH is its weight times that of weight 1, and so is its bound: a factor that is not a power of two
    adds one rounding, for which the bound of weight 1 holds four.  dW adds what its second factor loses: H times the row's weight
    over the largest such product, which ends at 2^-39 of that (two FP16 numbers, or one) and meets probabilities of weight 1."""
    g, hidden, weight, targets = _inputs(rows + width, rows, width, vocab, dtype, ignored)
    order = torch.randperm(rows, generator=g, device="cuda")
    upstream = (10.0**torch.linspace(lowest, highest, rows, device="cuda", dtype=torch.float64)).float()[order]
    upstream = upstream * torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    grads = _weighted(hidden, weight, targets, upstream, recompute)
    ones = torch.ones_like(upstream)
    values, bounds = reference.loss(hidden, weight, targets, -100, "none", ones, recompute)
    by = upstream.double()[:, None]
    assert_within("dH", grads[0], values[1] * by, bounds[1] * by.abs())
    values, bounds = reference.loss(hidden, weight, targets, -100, "none", upstream, recompute)
    kept = (targets != -100)[:, None]
    p = torch.softmax(hidden.double() @ weight.double().T, -1)
    p = (p + torch.nn.functional.one_hot(targets.clamp_min(0), vocab)) * kept
    largest = float((hidden.double().abs() * by.abs() * kept).max())
    assert_within("dW", grads[1], values[2], bounds[2] + 2.0**-39 * largest * p.sum(0)[:, None])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_a_row_is_the_same_beside_a_large_weight(dtype):
    """Powers of two as weights: the row's gradient is the same bits whatever the others weigh."""
    g, hidden, weight, targets = _inputs(5, 200, 160, 1000, dtype)
    alone = _weighted(hidden, weight, targets, torch.ones(200, device="cuda"), False)[0]
    upstream = torch.ones(200, device="cuda")
    upstream[17], upstream[90] = 2.0**40, 2.0**-30
    beside = _weighted(hidden, weight, targets, upstream, False)[0]
    others = (torch.arange(200, device="cuda") != 17) & (torch.arange(200, device="cuda") != 90)
    assert torch.equal(beside[others], alone[others])
    if dtype != FP16:
        assert torch.equal(beside[17], alone[17] * 2.0**40) and torch.equal(beside[90], alone[90] * 2.0**-30)


@pytest.mark.parametrize("dtype", [FP16, FP32])
def test_weighted_rows_captured_and_replayed(dtype):
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _, hidden, weight, targets = _inputs(9, 150, 64, 300, dtype)
        upstream = torch.ones(150, device="cuda")
        for _ in range(2):
            _weighted(hidden, weight, targets, upstream, False)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outputs = _weighted(hidden, weight, targets, upstream, False)
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        upstream.copy_(10.0**(-6 * torch.rand(150, generator=g, device="cuda")))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outputs]
        assert all(torch.equal(a, b) for a, b in zip(got, _weighted(hidden, weight, targets, upstream, False)))
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("recompute", [False, True])
def test_rows_of_no_weight_and_of_a_nonfinite_one(dtype, recompute):
    g, hidden, weight, targets = _inputs(7, 150, 64, 300, dtype)
    upstream = torch.ones(150, device="cuda")
    upstream[3] = 0.0
    grads = _weighted(hidden, weight, targets, upstream, recompute)
    assert not grads[0][3].any() and bool(grads[0].isfinite().all()) and bool(grads[1].isfinite().all())
    clean = grads[0]
    for bad in (float("nan"), float("inf")):
        upstream[40] = bad
        grads = _weighted(hidden, weight, targets, upstream, recompute)
        rows = torch.arange(150, device="cuda") != 40
        assert torch.equal(grads[0][rows], clean[rows])
        assert not bool(grads[0][40].isfinite().any()) and not bool(grads[1].isfinite().any())
    assert not _weighted(hidden, weight, targets, torch.zeros(150, device="cuda"), recompute)[1].any()


@pytest.mark.parametrize("dtype", [FP16, FP32])
def test_weights_of_rows_that_are_all_ignored(dtype):
    g, hidden, weight, targets = _inputs(11, 150, 64, 300, dtype)
    hidden[5] = float("nan")
    targets.fill_(-100)
    for recompute in (False, True):
        grads = _weighted(hidden, weight, targets, torch.full((150,), 1e6, device="cuda"), recompute)
        assert not grads[0].any() and not grads[1].any()
