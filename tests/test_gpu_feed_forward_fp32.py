"""FP32 inputs of the gated feed-forward block on the GPU: by FP32 instructions up to 1024 rows or
2^31 rows times widths, beyond as sums of three BF16 numbers; sizes on both sides, and strides of
which the offsets would leave 32 bits.  Bounds as in tests/feed_forward_reference.py."""

from __future__ import annotations

import pytest
import torch

from attnres import layers
from test_gpu_feed_forward import FP32, _check, _inputs, _run

pytestmark = pytest.mark.gpu

PARTS = (1056, 1056, 2048, 640)  # 1056 rows, 2.28e9 > 2^31 rows times widths


# rows, width, hidden, out_width
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("sizes", [(1024, 1024, 2112, 96), (1030, 1000, 2100, 1024), PARTS, (2051, 520, 330, 72), (3000, 8, 40, 2000),
                                   (20, 96, 8000, 33), (129, 2050, 64, 128), (48, 64, 4096, 192)])
def test_by_either_kind_of_product(sizes, activation):
    _check(*_inputs(31, *sizes, FP32), activation=activation)


def test_recomputed_and_one_by_one():
    x, gate_up, down, grad = _inputs(32, *PARTS, FP32)
    whole = _run(x, gate_up, down, grad)
    for kept, formed in zip(whole, _run(x, gate_up, down, grad, recompute=True)):
        assert torch.equal(kept, formed)
    for which in range(3):
        leaves = [t.detach().requires_grad_(i == which) for i, t in enumerate((x, gate_up, down))]
        (gradient,) = torch.autograd.grad(layers.gated_feed_forward(*leaves), leaves[which], grad)
        _values = whole[1 + which].double()
        # another cut of the depth at most: FP32 sums in another order
        assert float((gradient.double() - _values).norm() / _values.norm()) <= 2.0**-20


def test_over_the_exponents():
    x, gate_up, down, grad = _inputs(33, *PARTS, FP32)
    powers = torch.exp2(torch.arange(PARTS[0], device="cuda") % 48 * 2.0 - 48)[:, None]
    _check(x * 1e-3, gate_up, down * 2.0**60, grad * powers)


@pytest.mark.parametrize("sizes", [PARTS, (300, 1056, 2048, 640)])
def test_a_nonfinite_row_stays_in_its_own(sizes):
    x, gate_up, down, grad = _inputs(34, *sizes, FP32)
    clean = _run(x, gate_up, down, grad)
    x[7, 3], x[70, 4] = float("nan"), float("inf")
    out, dx, *_ = _run(x, gate_up, down, grad)
    others = torch.ones(sizes[0], dtype=torch.bool, device="cuda")
    others[[7, 70]] = False
    assert torch.equal(out[others], clean[0][others]) and torch.equal(dx[others], clean[1][others])
    assert bool(torch.isnan(out[7]).all()) and not bool(torch.isfinite(out[70]).any())


@pytest.mark.parametrize("hidden", [96, 192])  # times 2^22 elements: within and beyond 2^29 to the up projection's rows
def test_weights_far_apart(hidden):
    x, gate_up, down, grad = _inputs(35, 40, 64, hidden, 32, FP32)
    apart = torch.empty(2 * hidden, 2**22, device="cuda")[:, :64]
    apart.copy_(gate_up)
    for expected, actual in zip(_run(x, gate_up, down, grad), _run(x, apart, down, grad)):
        assert torch.equal(expected, actual)


@pytest.mark.parametrize("sizes", [PARTS, (700, 512, 1024, 512)])
def test_the_same_bits_captured_and_replayed(sizes):
    x, gate_up, down, _grad = _inputs(36, *sizes, FP32)
    with torch.no_grad():
        expected = layers.gated_feed_forward(x, gate_up, down)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layers.gated_feed_forward(x, gate_up, down)
        for scale in (2.0, 0.5):
            x.mul_(scale)
            graph.replay()
            assert torch.equal(out, layers.gated_feed_forward(x, gate_up, down))
        assert torch.equal(out, expected)
