"""The gated feed-forward block (attnres.layers) on the GPU against its FP64 definition
(tests/feed_forward_reference.py, where the bounds are derived): sizes around the edges
of the kernels' tiles and stages, types, layouts, what may be recomputed, streams and graphs."""

from __future__ import annotations

import pytest
import torch

import feed_forward_reference as reference
from attnres import attnres, layers
from layer_reference import assert_within

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("out", "dx", "dgate_up", "ddown")


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _inputs(seed, rows, width, hidden, out_width, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return ((_randn(g, rows, width) * torch.exp(_randn(g, rows, 1))).to(dtype), (_randn(g, 2 * hidden, width) * width**-0.5).to(dtype),
            (_randn(g, out_width, hidden) * hidden**-0.5).to(dtype), _randn(g, rows, out_width).to(dtype))


def _run(x, gate_up, down, grad, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (x, gate_up, down)]
    out = layers.gated_feed_forward(*leaves, **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, grad.reshape(out.shape)))


def _check(x, gate_up, down, grad, activation="silu", **kw):
    results = _run(x, gate_up, down, grad, activation=activation, **kw)
    values, bounds, norms = reference.feed_forward(x, gate_up, down, activation, grad)
    for name, actual, value, bound, norm, like in zip(NAMES, results, values, bounds, norms,
                                                      ((*x.shape[:-1], down.shape[0]), x.shape, gate_up.shape, down.shape)):
        assert actual.shape == torch.Size(like) and actual.dtype == x.dtype and actual.is_contiguous(), name
        flat = actual.reshape(value.shape)
        if x.dtype == FP16:  # what FP16 does not hold becomes an infinity
            limit = 65504.0 * (1 + 2.0**-11)
            beyond, near = value.abs() - bound > limit, value.abs() + bound >= limit
            assert torch.equal(flat[beyond].double(), value[beyond].sign() * float("inf")), name
            flat, value = flat.masked_fill(near, 0.0), value.masked_fill(near, 0.0)
        assert_within(name, flat, value, bound)
        if value.numel() >= 4096:
            off = float((flat.double() - value).norm() / value.norm())
            assert off <= norm, (name, off, norm)
    return results


# rows, width, hidden, out_width
SIZES = [(1, 1, 1, 1), (1, 64, 128, 64), (3, 7, 5, 9), (17, 32, 96, 32), (31, 33, 31, 65), (64, 128, 160, 96), (65, 96, 127, 160),
         (256, 256, 128, 256), (257, 264, 129, 257), (300, 512, 384, 130), (100, 1537, 700, 1000), (513, 100, 1030, 520),
         (1025, 320, 288, 64)]


@pytest.mark.parametrize("dtype,activation", [(BF16, "silu"), (BF16, "gelu"), (FP16, "silu"), (FP16, "gelu"), (FP32, "silu"), (FP32, "gelu")])
@pytest.mark.parametrize("rows,width,hidden,out_width", SIZES)
def test_feed_forward(rows, width, hidden, out_width, dtype, activation):
    _check(*_inputs(rows * 7 + width, rows, width, hidden, out_width, dtype), activation)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_the_widest_rows(dtype):
    _check(*_inputs(5, 70, 8192, 200, 8192, dtype))


def test_the_most_hidden_entries():
    _check(*_inputs(6, 33, 64, 65536, 32, BF16))


@pytest.mark.parametrize("rows", [2, 8, 15, 16, 18, 32, 33, 48, 63, 66, 128, 200])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_forward_alone_of_few_rows(rows, dtype):
    """Serving: no gradients.  The same definition, and rows do not depend on how many there are beyond their own bound."""
    x, gate_up, down, grad = _inputs(rows, rows, 320, 416, 192, dtype)
    values, bounds, _norms = reference.feed_forward(x, gate_up, down, "silu", grad)
    with torch.no_grad():
        out = layers.gated_feed_forward(x, gate_up, down)
    assert_within("out", out, values[0], bounds[0])
    assert not out.requires_grad


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_recomputed_gradients(dtype):
    inputs = _inputs(8, 200, 160, 224, 96, dtype)
    kept, again = _check(*inputs), _check(*inputs, recompute=True)
    assert all(torch.equal(a, b) for a, b in zip(kept, again))


@pytest.mark.parametrize("rows", [5, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_gradients_asked_for_one_by_one(rows, dtype):
    x, gate_up, down, grad = _inputs(9, rows, 96, 200, 64, dtype)
    together = _run(x, gate_up, down, grad)
    for wanted in range(3):
        leaves = [t.detach().requires_grad_(k == wanted) for k, t in enumerate((x, gate_up, down))]
        out = layers.gated_feed_forward(*leaves)
        (alone,) = torch.autograd.grad(out, leaves[wanted], grad)
        assert torch.equal(alone, together[1 + wanted])


@pytest.mark.parametrize("layout", ["rows_apart", "off_by_one", "transposed", "one_row_for_all", "batch_axes", "weights_apart"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_layouts(layout, dtype):
    rows, width, hidden, out_width = 96, 128, 160, 64
    x, gate_up, down, grad = _inputs(10, rows, width, hidden, out_width, dtype)
    if layout == "rows_apart":
        x = torch.nn.functional.pad(x, (8, 16), value=float("nan"))[:, 8:8 + width]
    elif layout == "off_by_one":
        x = torch.nn.functional.pad(x, (1, 3))[:, 1:1 + width]
        gate_up = torch.nn.functional.pad(gate_up, (3, 0))[:, 3:]
        down = torch.nn.functional.pad(down, (5, 1))[:, 5:5 + hidden]
        grad = torch.nn.functional.pad(grad.flatten(), (1, 0))[1:].view(rows, out_width)
    elif layout == "transposed":
        x, gate_up, down, grad = (t.T.contiguous().T for t in (x, gate_up, down, grad))
    elif layout == "one_row_for_all":
        x, grad = x[:1].expand(rows, width), grad[:1].expand(rows, out_width)
    elif layout == "batch_axes":
        x, grad = x.view(4, 3, 8, width), grad.view(4, 3, 8, out_width)
    else:
        gate_up = torch.nn.functional.pad(gate_up, (0, 64))[:, :width]
        down = torch.nn.functional.pad(down, (0, 0, 2, 2))[2:2 + out_width]
    _check(x, gate_up, down, grad)
    expected = _run(*(t.contiguous() for t in (x, gate_up, down, grad)))
    assert all(torch.equal(a, b) for a, b in zip(_run(x, gate_up, down, grad), expected))


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64)])
def test_no_rows(shape):
    x = torch.zeros(shape, device="cuda", dtype=BF16, requires_grad=True)
    gate_up, down = (torch.randn(s, device="cuda", dtype=BF16).requires_grad_(True) for s in ((256, 64), (32, 128)))
    out = layers.gated_feed_forward(x, gate_up, down)
    assert out.shape == (*shape[:-1], 32)
    grads = torch.autograd.grad(out.sum(), (x, gate_up, down))
    assert [g.shape for g in grads] == [x.shape, gate_up.shape, down.shape]
    assert not any(bool(g.any()) for g in grads)


def test_one_row_without_axes():
    x, gate_up, down, grad = _inputs(11, 1, 96, 64, 32, BF16)
    _check(x[0], gate_up, down, grad[0])


@pytest.mark.parametrize("rows", [33, 64, 300])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_a_nonfinite_row_stays_in_its_own(rows, dtype):
    """Of the rows' outputs and gradients; the last row too, which fills up the products' last stage."""
    inputs = _inputs(12, rows, 64, 96, 64, dtype)
    clean = _run(*inputs)
    for row in (0, rows - 1):
        for bad in (float("nan"), float("inf")):
            x, gate_up, down, grad = inputs
            x = x.clone()
            x[row, 3] = bad
            out, dx, *_ = _run(x, gate_up, down, grad)
            others = torch.arange(rows, device="cuda") != row
            assert torch.equal(out[others], clean[0][others]) and torch.equal(dx[others], clean[1][others])
            assert not bool(out[row].isfinite().all())
    x, gate_up, down, grad = inputs
    grad = grad.clone()
    grad[rows - 1, 0] = float("inf")
    out, dx, _dw, ddown = _run(x, gate_up, down, grad)
    others = torch.arange(rows, device="cuda") != rows - 1
    assert torch.equal(out, clean[0]) and torch.equal(dx[others], clean[1][others])
    assert torch.equal(ddown[1:], clean[3][1:]) and not bool(ddown[0].isfinite().any())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_large_and_small_projections(dtype, activation):
    """Gates far from zero on both sides, where the exponential leaves its type, and of zero."""
    rows, width = 64, 32
    x = torch.zeros(rows, width, device="cuda")
    x[:, 0] = torch.linspace(-100.0, 100.0, rows, device="cuda")
    x[32, 0] = 0.0
    x[:, 1] = 1.0
    gate_up = torch.zeros(128, width, device="cuda")
    gate_up[:64, 0] = torch.linspace(-1.5, 1.5, 64, device="cuda")
    gate_up[64:, 1] = torch.linspace(0.5, 2.0, 64, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(13)
    _check(x.to(dtype), gate_up.to(dtype), _randn(g, 32, 64).to(dtype), _randn(g, rows, 32).to(dtype), activation)


def test_fp32_over_the_exponents():
    """FP32 keeps its 24 bits over its range: rows and weights of very different magnitudes."""
    x, gate_up, down, grad = _inputs(14, 96, 64, 64, 64, FP32)
    powers = torch.exp2(torch.arange(96, device="cuda") % 48 * 2.0 - 48)[:, None]
    _check(x * 1e-3, gate_up, down * 2.0**60, grad * powers)


def test_gradients_against_differences():
    x, gate_up, down, grad = (t.double() for t in _inputs(15, 12, 32, 48, 16, FP32))
    _out, *grads = _run(*(t.float() for t in (x, gate_up, down, grad)))
    g = torch.Generator(device="cuda").manual_seed(16)
    for which, gradient in enumerate(grads):
        direction = _randn(g, *gradient.shape).double()
        step = 1e-2

        def value(sign):
            leaves = [x, gate_up, down]
            leaves[which] = leaves[which] + sign * step * direction
            return float((layers.gated_feed_forward(*(t.float() for t in leaves)).double() * grad).sum())

        by_difference = (value(1) - value(-1)) / (2 * step)
        expected = float((gradient.double() * direction).sum())
        # the third derivative's term, step^2 / 6 of it, and FP32's rounding over the step
        scale = float((gradient.double().abs() * direction.abs()).sum())
        assert abs(by_difference - expected) <= 1e-2 * scale, which


def test_repeated_calls_give_the_same_bits():
    inputs = _inputs(17, 700, 512, 640, 256, BF16)
    first = _run(*inputs)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(_run(*inputs), first))


def test_another_stream_and_a_graph_kept_for_a_second_backward():
    x, gate_up, down, grad = _inputs(18, 300, 256, 320, 128, BF16)
    expected = _run(x, gate_up, down, grad)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        leaves = [t.detach().requires_grad_(True) for t in (x, gate_up, down)]
        out = layers.gated_feed_forward(*leaves)
        first = torch.autograd.grad(out, leaves, grad, retain_graph=True)
        second = torch.autograd.grad(out, leaves, grad)
    stream.synchronize()
    for grads in (first, second):
        assert all(torch.equal(a, b) for a, b in zip((out.detach(), *grads), expected))


@pytest.mark.parametrize("rows,dtype", [(1, BF16), (24, FP32), (300, BF16), (300, FP32), (64, FP16)])
def test_captured_and_replayed(rows, dtype):
    """Two graphs with workspaces of their own, replayed with eager work between the replays and once at the same time."""
    graphs, streams = [], []
    for seed in (19, 20):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            static = [t.detach().clone().requires_grad_(k < 3) for k, t in enumerate(_inputs(seed, rows, 96, 160, 64, dtype))]

            def step(static=static):
                out = layers.gated_feed_forward(*static[:3])
                return (out.detach(), *torch.autograd.grad(out, static[:3], static[3]))

            step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            results = step()
        graphs.append((graph, static, results))
        streams.append(stream)
    for round in range(3):
        expected = []
        for k, (graph, static, results) in enumerate(graphs):
            fresh = _inputs(100 * round + k, rows, 96, 160, 64, dtype)
            with torch.no_grad():
                for to, value in zip(static, fresh):
                    to.copy_(value)
            expected.append(_run(*fresh))
            torch.cuda.synchronize()
        for (graph, _static, _results), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_graph, _static, results), want in zip(graphs, expected):
            assert all(torch.equal(a, b) for a, b in zip(results, want))


def test_compiled_matches_eager():
    x, gate_up, down, grad = _inputs(21, 60, 96, 160, 64, BF16)

    def forward(x, gate_up, down):
        return layers.gated_feed_forward(x, gate_up, down, activation="gelu") * 2

    compiled = torch.compile(forward, fullgraph=True, backend="aot_eager")
    results = []
    for call in (forward, compiled):
        leaves = [t.detach().requires_grad_(True) for t in (x, gate_up, down)]
        out = call(*leaves)
        results.append((out.detach(), *torch.autograd.grad(out, leaves, grad)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    with torch.no_grad():
        assert torch.equal(compiled(x, gate_up, down), results[0][0])


def test_compiled_for_any_number_of_rows():
    _x, gate_up, down, _grad = _inputs(27, 1, 96, 160, 64, BF16)
    gate_up.requires_grad_(True), down.requires_grad_(True)
    compiled = torch.compile(lambda x: layers.gated_feed_forward(x, gate_up, down), fullgraph=True, backend="aot_eager", dynamic=True)
    for rows in (3, 40, 200):
        x, _gate_up, _down, grad = _inputs(28, rows, 96, 160, 64, BF16)
        results = []
        for call in (compiled, lambda x: layers.gated_feed_forward(x, gate_up, down)):
            leaf = x.detach().requires_grad_(True)
            out = call(leaf)
            results.append((out.detach(), *torch.autograd.grad(out, (leaf, gate_up, down), grad)))
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_checkpointed():
    """The forward again in the backward gives the bits of the first one, few rows or many."""
    from torch.utils.checkpoint import checkpoint

    for rows in (5, 60, 300):
        x, gate_up, down, grad = _inputs(29, rows, 96, 160, 64, BF16)
        results = []
        for call in (lambda *t: checkpoint(layers.gated_feed_forward, *t, use_reentrant=False), layers.gated_feed_forward):
            leaves = [t.detach().requires_grad_(True) for t in (x, gate_up, down)]
            out = call(*leaves)
            results.append((out.detach(), *torch.autograd.grad(out, leaves, grad)))
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_on_two_streams_at_once():
    inputs = [_inputs(30 + k, 700, 256, 512, 256, BF16) for k in range(2)]
    expected = [_run(*i) for i in inputs]
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in inputs], [[], []]
    for _ in range(3):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[k].append(_run(*inputs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for result in results[k]:
            assert all(torch.equal(a, b) for a, b in zip(result, expected[k]))


def test_differentiating_the_gradients_again_is_refused():
    x, gate_up, down, _grad = _inputs(22, 8, 32, 32, 32, BF16)
    x.requires_grad_(True)
    (grad,) = torch.autograd.grad(layers.gated_feed_forward(x, gate_up, down).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="first-order"):
        grad.square().sum().backward()


def test_tangents_are_refused():
    x, gate_up, down, _grad = _inputs(23, 8, 32, 32, 32, BF16)
    from torch.autograd import forward_ad

    for which in range(3):
        for grad in (False, True):
            with forward_ad.dual_level():
                leaves = [t.detach().requires_grad_(grad) for t in (x, gate_up, down)]
                leaves[which] = forward_ad.make_dual(leaves[which], torch.ones_like(leaves[which]))
                with pytest.raises(RuntimeError, match="forward|jvp"):
                    layers.gated_feed_forward(*leaves)


def test_inputs_changed_before_the_backward_are_refused():
    x, gate_up, down, grad = _inputs(24, 8, 32, 32, 32, BF16)
    gate_up.requires_grad_(True)
    out = layers.gated_feed_forward(x, gate_up, down)
    down.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(out, gate_up, grad)


def test_between_a_read_and_a_norm():
    """As a model runs it: a read, its norm, the block, and the next read of what it emits."""
    g = torch.Generator(device="cuda").manual_seed(25)
    sources = [_randn(g, 2, 24, 64).to(BF16).requires_grad_(True) for _ in range(2)]
    query = _randn(g, 64).to(BF16).requires_grad_(True)
    weight, bias = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    _x, gate_up, down, _grad = _inputs(26, 1, 64, 96, 64, BF16)
    gate_up.requires_grad_(True), down.requires_grad_(True)
    leaves = [*sources, query, weight, bias, gate_up, down]

    def plain(x):
        gate, up = (x.float() @ gate_up.float().T).chunk(2, -1)
        return ((torch.nn.functional.silu(gate) * up) @ down.float().T).to(BF16)

    results = []
    for block in (lambda x: layers.gated_feed_forward(x, gate_up, down), plain):
        emitted = block(layers.layer_norm(attnres(sources, query), weight, bias))
        out = attnres([*sources, emitted], query)
        results.append([out.detach(), *torch.autograd.grad(out.float().square().sum(), leaves)])
    for a, b in zip(*results):
        # a few roundings to BF16 apart: 2^-8 each, of `a`, its gradients and the results
        assert float((a.float() - b.float()).norm()) <= 4 * 2.0**-8 * float(b.float().norm())
