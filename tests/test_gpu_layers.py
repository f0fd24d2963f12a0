"""The layers around the reads (attnres.layers) on the GPU against their FP64
definitions (tests/layer_reference.py, where the bounds are derived): sizes
around every edge of the kernels' tiles, types, layouts, masks, and what lies in
masked places."""

from __future__ import annotations

import pytest
import torch

import layer_reference as reference
from attnres import _native, layers
from layer_reference import assert_within

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NAN = float("nan")


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


# --------------------------------------------------------------- layer norm

def _check_norm(x, weight, bias, grad, eps=1e-5):
    leaves = [t.requires_grad_(True) for t in (x, weight, bias) if t is not None]
    out = layers.layer_norm(x, weight, bias, eps=eps)
    assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous()
    grads = torch.autograd.grad(out, leaves, grad)
    wanted = [True, True, weight is not None, bias is not None]
    with torch.no_grad():
        values, bounds = reference.layer_norm(x, weight, bias, eps, grad)
        forward_only = layers.layer_norm(x, weight, bias, eps=eps)
    assert torch.equal(forward_only, out.detach()) or bool(out.isnan().any())
    names = [n for n, w in zip(("out", "dx", "dw", "db"), wanted) if w]
    for name, actual, value, bound in zip(names, (out.detach(), *grads),
                                          [v for v, w in zip(values, wanted) if w], [b for b, w in zip(bounds, wanted) if w]):
        assert_within(name, actual, value, bound)


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 2048), (3, 7), (65, 128), (31, 129), (17, 511), (40, 1024), (9, 1025),
                                        (700, 1537), (33, 2048), (5, 2049), (12, 4096), (3, 4097), (4, 6144), (3, 6145), (5, 8192)])
@pytest.mark.parametrize("dtype,params", [(BF16, FP32), (BF16, BF16), (FP16, FP16), (FP32, FP32)])
def test_layer_norm(rows, width, dtype, params):
    g = _generator(rows * 10007 + width)
    x = (_randn(g, rows, width) + 0.5 * _randn(g, width)).to(dtype)
    _check_norm(x, (1 + 0.2 * _randn(g, width)).to(params), (0.1 * _randn(g, width)).to(params), _randn(g, rows, width).to(dtype))


@pytest.mark.parametrize("has_weight,has_bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("width", [96, 1000, 3001])
def test_layer_norm_without_parameters(width, has_weight, has_bias):
    g = _generator(width)
    x = _randn(g, 2, 19, width).to(BF16)
    _check_norm(x, _randn(g, width) if has_weight else None, _randn(g, width) if has_bias else None,
                _randn(g, 2, 19, width).to(BF16))


def test_layer_norm_many_rows():
    """More rows than the backward's workgroups take at once."""
    g = _generator(5)
    for rows, width in ((9000, 64), (5000, 1024), (3000, 2048)):
        x = _randn(g, rows, width).to(BF16)
        _check_norm(x, _randn(g, width), _randn(g, width), _randn(g, rows, width).to(BF16))


@pytest.mark.parametrize("rows,width,dtype", [(20001, 3331, BF16), (9000, 4099, FP32)])
def test_layer_norm_of_results_past_the_caches(rows, width, dtype):
    """Results of more than 128 MiB, of rows that no store is aligned to."""
    g = _generator(rows)
    x = _randn(g, rows, width).to(dtype)
    _check_norm(x, _randn(g, width), _randn(g, width), _randn(g, rows, width).to(dtype))


@pytest.mark.parametrize("layout", ["slice", "offset", "transposed", "expanded", "vector", "steps"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_layer_norm_layouts(layout, dtype):
    g = _generator(11)
    wide = _randn(g, 6, 5, 515).to(dtype)
    x = {"slice": wide[..., :509], "offset": wide[1:, :, 3:300], "transposed": wide.transpose(0, 2),
         "expanded": wide[:1, :1].expand(4, 3, 515), "vector": wide[2, 3], "steps": wide[..., ::2]}[layout].detach()
    width = x.shape[-1]
    grad = _randn(g, width, *x.shape[:-1]).to(dtype).movedim(0, -1)  # a gradient that is not contiguous
    _check_norm(x, _randn(g, 2 * width)[::2], _randn(g, width), grad)


def test_layer_norm_rows_without_spread_and_with_an_offset():
    g = _generator(13)
    x = torch.cat([torch.full((2, 640), 3.0, device="cuda"), torch.zeros(1, 640, device="cuda"),
                   1000.0 + _randn(g, 3, 640), 1e-4 * _randn(g, 2, 640)])
    _check_norm(x, _randn(g, 640), _randn(g, 640), _randn(g, 8, 640))


def test_layer_norm_nonfinite_rows_stay_in_their_own():
    g = _generator(17)
    x, weight, bias = _randn(g, 9, 1024).to(BF16), _randn(g, 1024), _randn(g, 1024)
    clean = layers.layer_norm(x, weight, bias)
    x[2, 5], x[6, 1000] = NAN, float("inf")
    out = layers.layer_norm(x, weight, bias)
    keep = torch.tensor([0, 1, 3, 4, 5, 7, 8], device="cuda")
    assert torch.equal(out[keep], clean[keep])
    assert bool(out[[2, 6]].isnan().all(-1).all())


@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 640)])
def test_layer_norm_without_rows(shape):
    x = torch.empty(shape, device="cuda", dtype=BF16, requires_grad=True)
    weight = torch.ones(shape[-1], device="cuda", requires_grad=True)
    bias = torch.ones(shape[-1], device="cuda", requires_grad=True)
    out = layers.layer_norm(x, weight, bias)
    grads = torch.autograd.grad(out, (x, weight, bias), torch.empty_like(out))
    assert out.shape == x.shape and grads[0].shape == x.shape
    assert not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("wanted", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
def test_layer_norm_gradients_asked_for_one_by_one(wanted):
    g = _generator(19)
    inputs = [_randn(g, 50, 777).to(BF16), _randn(g, 777), _randn(g, 777)]
    grad = _randn(g, 50, 777).to(BF16)
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    everything = torch.autograd.grad(layers.layer_norm(*leaves), leaves, grad)
    some = [t.clone().requires_grad_(w) for t, w in zip(inputs, wanted)]
    got = torch.autograd.grad(layers.layer_norm(*some), [t for t, w in zip(some, wanted) if w], grad)
    for a, b in zip(got, [e for e, w in zip(everything, wanted) if w]):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- embedding

def _check_embedding(tokens, weight, positions, scale, dtype, seed=1):
    g = _generator(seed)
    leaves = [t.requires_grad_(True) for t in (weight, positions) if t is not None]
    out = layers.embedding(tokens, weight, positions, scale=scale, dtype=dtype)
    assert out.dtype == dtype and out.shape == (*tokens.shape, weight.shape[1])
    grad = _randn(g, *out.shape).to(dtype)
    grads = torch.autograd.grad(out, leaves, grad)
    with torch.no_grad():
        values, bounds = reference.embedding(tokens, weight, positions, scale, grad)
    for name, actual, value, bound in zip(("out", "dW", "dpos"), (out.detach(), *grads), values, bounds):
        assert_within(name, actual, value, bound)
    again = torch.autograd.grad(layers.embedding(tokens, weight, positions, scale=scale, dtype=dtype), leaves, grad)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("batch,length,vocab,width", [
    (1, 1, 1, 1), (1, 1, 5, 2048), (2, 7, 11, 5), (3, 64, 50, 65), (1, 2047, 1023, 72), (1, 2049, 1024, 8), (2, 1024, 1025, 1000),
    (4, 1030, 32768, 64), (1, 9000, 3, 129), (5, 3001, 70001, 16), (2, 33, 2000003, 8), (2, 5, 7, 8192)])
@pytest.mark.parametrize("table,dtype", [(BF16, BF16), (FP32, BF16), (FP16, FP32), (FP32, FP32)])
def test_embedding(batch, length, vocab, width, table, dtype):
    g = _generator(batch * length + vocab)
    tokens = (torch.rand(batch, length, generator=g, device="cuda")**3 * vocab).long().clamp_(0, vocab - 1)
    _check_embedding(tokens, _randn(g, vocab, width).to(table), _randn(g, length + 3, width).to(table), 1.5, dtype)


@pytest.mark.parametrize("length", [3, 64, 257, 5000])
def test_embedding_one_token_for_all(length):
    """One run of the sorted list across every piece, at both ends of the table."""
    g = _generator(length)
    for token in (0, 96):
        _check_embedding(torch.full((2, length), token, device="cuda"), _randn(g, 97, 40).to(BF16), None, 1.0, BF16)


@pytest.mark.parametrize("run", [1, 3, 4, 5, 8, 63, 64, 65, 200])
def test_embedding_runs_of_one_length(run):
    """Runs that end before, at and after the borders of the pieces."""
    g = _generator(run)
    tokens = torch.arange(4096, device="cuda") // run
    _check_embedding(tokens[torch.randperm(4096, generator=g, device="cuda")], _randn(g, 4100, 24), None, 2.0, FP32)


@pytest.mark.parametrize("length,vocab", [(48 * 1024, 500), (48 * 1024 + 1, 500), (70001, 3), (70001, 40000), (200000, 1500000)])
def test_embedding_of_many_tokens(length, vocab):
    """Around the number of tiles from which their counts are scanned by a launch of its own."""
    g = _generator(length)
    tokens = (torch.rand(length, generator=g, device="cuda")**2 * vocab).long().clamp_(0, vocab - 1)
    tokens[5::1000] = vocab  # outside
    _check_embedding(tokens, _randn(g, vocab, 16).to(BF16), None, 1.0, FP32)


def test_embedding_of_more_rows_than_a_launch_has_groups():
    """8 threads to a row: more than 2^32 of them."""
    g = _generator(53)
    weight = _randn(g, 1000, 1).to(BF16)
    tokens = torch.randint(1000, (2**29,), generator=g, device="cuda", dtype=torch.int32)
    out = layers.embedding(tokens, weight)
    for part, ids in zip(out[:, 0].split(2**26), tokens.split(2**26)):
        assert torch.equal(part, weight[:, 0].take(ids.long()))


def test_embedding_integer_types_batches_and_layouts():
    g = _generator(23)
    weight, positions = _randn(g, 300, 96).to(BF16), _randn(g, 40, 96).to(BF16)
    tokens = torch.randint(300, (3, 2, 40), generator=g, device="cuda")
    _check_embedding(tokens.int(), weight.clone(), positions.clone(), 1.0, BF16)
    _check_embedding(tokens.transpose(0, 1), weight.clone(), positions.clone(), -0.25, BF16)
    _check_embedding(tokens[..., ::3], weight.clone(), None, 1.0, FP32)
    _check_embedding(tokens[0, 0], _randn(g, 96, 300).T.detach(), None, 1.0, FP32)


def test_embedding_tokens_outside_the_table():
    g = _generator(29)
    tokens = torch.randint(64, (2, 500), generator=g, device="cuda")
    tokens[0, ::7] = 64
    tokens[1, ::5] = -1
    tokens[1, 3] = 2**40
    _check_embedding(tokens, _randn(g, 64, 200).to(BF16), None, 1.0, BF16)
    everything = torch.full((1, 300), -100, device="cuda")
    _check_embedding(everything, _randn(g, 64, 200).to(BF16), None, 1.0, BF16)


def test_embedding_without_tokens():
    weight = torch.ones(10, 64, device="cuda", requires_grad=True)
    positions = torch.ones(4, 64, device="cuda", requires_grad=True)
    for shape in ((0, 3), (2, 0)):
        tokens = torch.empty(shape, device="cuda", dtype=torch.int64)
        out = layers.embedding(tokens, weight, positions)
        grads = torch.autograd.grad(out, (weight, positions), torch.empty_like(out))
        assert out.shape == (*shape, 64) and not grads[0].any() and not grads[1].any()


# --------------------------------------------------------------------- loss

def _loss_inputs(seed, rows, width, vocab, dtype, ignored=0.0):
    g = _generator(seed)
    hidden = _randn(g, rows, width).to(dtype)
    weight = (_randn(g, vocab, width) * (2.0 / width**0.5)).to(dtype)
    targets = torch.randint(vocab, (rows,), generator=g, device="cuda")
    targets[torch.rand(rows, generator=g, device="cuda") < ignored] = -100
    return g, hidden, weight, targets


def _check_loss(hidden, weight, targets, reduction, g, ignore_index=-100, recompute=False):
    leaves = (hidden.requires_grad_(True), weight.requires_grad_(True))
    out = layers.linear_cross_entropy(*leaves, targets, ignore_index=ignore_index, reduction=reduction, recompute=recompute)
    assert out.dtype == FP32 and out.shape == (targets.shape if reduction == "none" else ())
    grad = _randn(g, *out.shape) if out.dim() else _randn(g, 1)[0]
    grads = torch.autograd.grad(out, leaves, grad)
    with torch.no_grad():
        values, bounds = reference.loss(hidden, weight, targets, ignore_index, reduction, grad, recompute)
        scored = layers.linear_cross_entropy(*leaves, targets, ignore_index=ignore_index, reduction=reduction)
    assert torch.equal(scored, out.detach()) or bool(out.isnan().any())
    for name, actual, value, bound in zip(("loss", "dH", "dW"), (out.detach(), *grads), values, bounds):
        assert_within(name, actual, value, bound)


@pytest.mark.parametrize("rows,width,vocab", [(1, 1, 1), (1, 64, 17), (5, 7, 3), (2, 128, 256), (255, 65, 257), (256, 64, 256),
                                              (257, 100, 1000), (300, 1000, 513), (16, 1024, 5001), (600, 320, 2049),
                                              (70, 4096, 300), (33, 8192, 129), (1500, 24, 96)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("recompute", [False, True])
def test_loss(rows, width, vocab, dtype, recompute):
    g, hidden, weight, targets = _loss_inputs(rows + width + vocab, rows, width, vocab, dtype)
    _check_loss(hidden, weight, targets, "mean", g, recompute=recompute)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("ignored", [0.3, 0.95])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("recompute", [False, True])
def test_loss_with_ignored_targets(reduction, ignored, dtype, recompute):
    g, hidden, weight, targets = _loss_inputs(31, 700, 200, 900, dtype, ignored)
    _check_loss(hidden, weight, targets, reduction, g, recompute=recompute)


@pytest.mark.parametrize("recompute", [False, True])
def test_loss_in_several_pieces_of_the_vocabulary(recompute):
    """More probabilities than are formed at once."""
    g, hidden, weight, targets = _loss_inputs(37, 4096, 64, 70001, BF16, 0.1)
    _check_loss(hidden, weight, targets, "mean", g, recompute=recompute)


def test_loss_fp32_in_several_pieces_of_the_vocabulary():
    g, hidden, weight, targets = _loss_inputs(39, 1900, 40, 70001, FP32, 0.1)
    _check_loss(hidden, weight, targets, "none", g)


@pytest.mark.parametrize("rows", [15, 16, 17, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_loss_around_the_forward_of_few_rows(rows, dtype):
    for width, vocab, ignored in ((72, 63, 0.0), (1000, 130, 0.5)):
        g, hidden, weight, targets = _loss_inputs(rows + width, rows, width, vocab, dtype, ignored)
        _check_loss(hidden, weight, targets, "none", g)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("recompute", [False, True])
def test_loss_of_few_rows(reduction, dtype, recompute):
    """Rows that lie apart, ignored ones that hold NaN, one gradient at a time, the same graph twice."""
    for rows, width, vocab in ((3, 1000, 257), (20, 333, 2049), (32, 256, 31), (50, 77, 700), (17, 72, 16500)):
        g, hidden, weight, targets = _loss_inputs(67 + rows, rows, width, vocab, dtype, 0.4)
        wide = torch.full((rows, width + 5), NAN, device="cuda", dtype=dtype)
        wide[:, 2:width + 2] = torch.where((targets == -100)[:, None], torch.full_like(hidden, NAN), hidden)
        hidden = wide[:, 2:width + 2]
        _check_loss(hidden, weight, targets, reduction, g, recompute=recompute)
        h, w = hidden.detach().requires_grad_(True), weight.detach().requires_grad_(True)
        out = layers.linear_cross_entropy(h, w, targets, reduction=reduction, recompute=recompute)
        both = torch.autograd.grad(out, (h, w), torch.ones_like(out), retain_graph=True)
        again = torch.autograd.grad(out, (h, w), torch.ones_like(out))
        assert all(torch.equal(a, b) for a, b in zip(both, again))
        for k, leaf in enumerate((h, w)):
            alone = (h if k == 0 else h.detach(), w if k == 1 else w.detach())
            out = layers.linear_cross_entropy(*alone, targets, reduction=reduction, recompute=recompute)
            (one,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
            assert torch.equal(one, both[k])


def test_loss_of_few_rows_marks_a_target_outside_the_vocabulary():
    for recompute in (False, True):
        g, hidden, weight, targets = _loss_inputs(71, 12, 96, 200, BF16)
        targets[5] = 200
        hidden.requires_grad_(True), weight.requires_grad_(True)
        out = layers.linear_cross_entropy(hidden, weight, targets, reduction="none", recompute=recompute)
        grad_hidden, grad_weight = torch.autograd.grad(out, (hidden, weight), torch.ones_like(out))
        bad = torch.arange(12, device="cuda") == 5
        assert torch.equal(out.isnan(), bad) and torch.equal(grad_hidden.isnan().all(-1), bad)
        assert bool(grad_hidden[~bad].isfinite().all()) and bool(grad_weight.isnan().all())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_loss_graph_kept_for_a_second_backward(dtype):
    g, hidden, weight, targets = _loss_inputs(73, 400, 128, 1000, dtype, 0.2)
    hidden.requires_grad_(True), weight.requires_grad_(True)
    out = layers.linear_cross_entropy(hidden, weight, targets)
    first = torch.autograd.grad(out, (hidden, weight), retain_graph=True)
    second = torch.autograd.grad(out, (hidden, weight))
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_loss_of_one_token_without_axes():
    g, hidden, weight, targets = _loss_inputs(40, 1, 64, 50, BF16)
    _check_loss(hidden[0].detach(), weight, targets[0], "mean", g)


def test_loss_of_no_targets():
    g, hidden, weight, targets = _loss_inputs(41, 300, 64, 500, BF16)
    targets.fill_(-100)
    hidden.requires_grad_(True), weight.requires_grad_(True)
    for reduction, value in (("mean", NAN), ("sum", 0.0), ("none", 0.0)):
        out = layers.linear_cross_entropy(hidden, weight, targets, reduction=reduction)
        grads = torch.autograd.grad(out, (hidden, weight), torch.ones_like(out))
        assert bool((out.isnan() if value != value else out == value).all())
        assert not grads[0].any() and not grads[1].any()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_loss_does_not_look_at_ignored_rows(dtype):
    g, hidden, weight, targets = _loss_inputs(43, 520, 128, 777, dtype, 0.4)
    masked = targets == -100
    hidden[masked] = torch.where(torch.rand(int(masked.sum()), 128, generator=g, device="cuda") < 0.5, NAN, float("inf")).to(dtype)
    hidden[masked.nonzero()[0]] = torch.finfo(dtype).max
    for recompute in (False, True):
        _check_loss(hidden.detach(), weight.detach(), targets, "none", g, recompute=recompute)


def test_loss_of_a_nonfinite_row_stays_in_its_own():
    g, hidden, weight, targets = _loss_inputs(47, 300, 128, 600, BF16)
    clean = layers.linear_cross_entropy(hidden, weight, targets, reduction="none")
    hidden[7, 3] = NAN
    out = layers.linear_cross_entropy(hidden, weight, targets, reduction="none")
    keep = torch.arange(300, device="cuda") != 7
    assert torch.equal(out[keep], clean[keep]) and bool(out[7].isnan())


@pytest.mark.parametrize("recompute", [False, True])
def test_loss_marks_a_target_outside_the_vocabulary(recompute):
    g, hidden, weight, targets = _loss_inputs(53, 300, 128, 600, BF16)
    clean = layers.linear_cross_entropy(hidden, weight, targets, reduction="none")
    targets[4], targets[9], targets[200] = 600, -1, 2**33
    hidden.requires_grad_(True), weight.requires_grad_(True)
    out = layers.linear_cross_entropy(hidden, weight, targets, reduction="none", recompute=recompute)
    bad = torch.zeros(300, device="cuda", dtype=torch.bool)
    bad[[4, 9, 200]] = True
    assert torch.equal(out.isnan(), bad) and torch.equal(out[~bad], clean[~bad])
    grad_hidden, grad_weight = torch.autograd.grad(out, (hidden, weight), torch.ones_like(out))
    assert bool(grad_hidden[bad].isnan().all()) and bool(grad_hidden[~bad].isfinite().all())
    assert bool(grad_weight.isnan().all())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_loss_of_large_logits(dtype):
    """Logits of +-2000: certain rows have a loss of 0 to rounding, wrong ones thousands."""
    g, hidden, weight, targets = _loss_inputs(59, 200, 64, 300, dtype)
    with torch.no_grad():
        hidden.mul_(300.0)
        targets[:100] = (hidden[:100].float() @ weight.float().T).argmax(-1)
    for recompute in (False, True):
        _check_loss(hidden.detach(), weight.detach(), targets, "none", g, recompute=recompute)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_loss_of_huge_logits(dtype):
    """Logits beyond 2^24, whose neighbours are more than 1 apart: rows of equal logits, whose losses are log V, and rows whose
    target's logit is the largest, whose losses are 0.  Bounds: a few roundings of numbers up to 16."""
    hidden = torch.tensor([[0.0, 2.0**26], [2.0**26, 0.0]], device="cuda").to(dtype).repeat(40, 1)
    weight = torch.stack((torch.linspace(-8, 8, 300, device="cuda").to(dtype), torch.ones(300, device="cuda", dtype=dtype)), 1)
    targets = torch.full((80,), 299, device="cuda")
    for recompute in (False, True):
        h, w = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        out = layers.linear_cross_entropy(h, w, targets, reduction="none", recompute=recompute)
        (grad,) = torch.autograd.grad(out, h, torch.ones_like(out))
        assert bool((out[0::2] - torch.tensor(300.0).log().cuda()).abs().max() <= 2.0**-18)
        assert bool((out[1::2] >= 0).all()) and bool(out[1::2].max() <= 2.0**-18)
        # P of the second kind of rows is 0 but for roundings of its one entry, 1 - 1: 2^-8 of weights up to 8
        assert bool(grad[1::2].abs().max() <= 8 * (2.0**-8 if dtype == BF16 else 2.0**-20))


@pytest.mark.parametrize("scale_h,scale_w", [(1e-6, 1.0), (1e-20, 1e18), (1e12, 1e-13), (0.0, 1.0), (1.0, 0.0)])
def test_loss_fp32_over_the_exponents(scale_h, scale_w):
    g, hidden, weight, targets = _loss_inputs(61, 130, 96, 400, FP32)
    for recompute in (False, True):
        _check_loss(hidden * scale_h, weight * scale_w, targets, "sum", g, recompute=recompute)


@pytest.mark.parametrize("layout", ["slices", "misaligned", "transposed", "batched", "columns"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_loss_layouts(layout, dtype):
    g = _generator(67)
    h, w = _randn(g, 4, 60, 400).to(dtype), (0.2 * _randn(g, 512, 400)).to(dtype)
    hidden, weight = {"slices": (h[..., 8:136], w[::2, 8:136]), "misaligned": (h[..., 1:129], w[:, 3:131]),
                      "transposed": (h.transpose(0, 1)[..., :128], w[:128, :128].T), "batched": (h[..., :320], w[:, :320]),
                      "columns": (h[..., ::2], w[:, 1::2])}[layout]
    targets = torch.randint(weight.shape[0], (hidden.shape[1], hidden.shape[0]), generator=g, device="cuda").T.int()
    _check_loss(hidden.detach(), weight.detach(), targets, "none", g)


def test_loss_other_ignore_index_and_a_target_equal_to_it():
    g, hidden, weight, targets = _loss_inputs(71, 300, 64, 50, BF16)
    _check_loss(hidden, weight, targets, "mean", g, ignore_index=7)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("which", [0, 1])
def test_loss_gradients_asked_for_one_by_one(dtype, which):
    g, hidden, weight, targets = _loss_inputs(73, 300, 192, 1000, dtype, 0.2)
    leaves = [hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)]
    both = torch.autograd.grad(layers.linear_cross_entropy(*leaves, targets), leaves)
    one = [hidden.clone(), weight.clone()]
    one[which].requires_grad_(True)
    (got,) = torch.autograd.grad(layers.linear_cross_entropy(*one, targets), one[which])
    assert torch.equal(got, both[which])


def test_loss_without_rows():
    hidden = torch.empty(0, 64, device="cuda", dtype=BF16, requires_grad=True)
    weight = torch.ones(10, 64, device="cuda", dtype=BF16, requires_grad=True)
    targets = torch.empty(0, device="cuda", dtype=torch.int64)
    for reduction in ("none", "sum", "mean"):
        out = layers.linear_cross_entropy(hidden, weight, targets, reduction=reduction)
        grads = torch.autograd.grad(out, (hidden, weight), torch.ones_like(out))
        assert grads[0].shape == hidden.shape and not grads[1].any()
        assert out.numel() == 0 if reduction == "none" else bool(out.isnan() if reduction == "mean" else out == 0)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_loss_without_rows_through_the_c_abi(dtype):
    lib = _native.load()
    vocab, width, mean = 300, 40, 2
    weight = _randn(_generator(6), vocab, width).to((BF16, FP16, FP32)[dtype])
    saved = torch.empty(lib.attnres_hip_loss_saved_bytes(0, vocab, width, dtype, 1), dtype=torch.uint8, device="cuda")
    loss, grad = torch.zeros((), device="cuda"), torch.ones((), device="cuda")
    grad_weight = torch.full_like(weight, 7.0)
    stream = torch.cuda.current_stream().cuda_stream
    for backward in (0, 1):
        size = lib.attnres_hip_loss_workspace_bytes(0, vocab, width, dtype, 1, backward)
        workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
        if backward:
            status = lib.attnres_hip_loss_backward(None, width, weight.data_ptr(), width, 0, vocab, width, dtype, mean, 1,
                                                   saved.data_ptr(), grad.data_ptr(), None, grad_weight.data_ptr(),
                                                   workspace.data_ptr(), size, stream)
        else:
            status = lib.attnres_hip_loss_forward(None, width, weight.data_ptr(), width, None, 8, 0, vocab, width, dtype, -100,
                                                  mean, 1, loss.data_ptr(), saved.data_ptr(), workspace.data_ptr(), size, stream)
        assert status == 0, lib.attnres_hip_last_error().decode()
    assert bool(loss.isnan()) and not grad_weight.any()


def test_loss_gradient_against_differences():
    """The slope of the loss along its own gradient, by central differences.  What the step's width
    leaves out is taken from the definition in FP64 (its differences against its derivative); the two FP32
    losses, about 7, are off by at most 1e-5 each (their bound at this size is 2e-6)."""
    g, hidden, weight, targets = _loss_inputs(79, 64, 96, 200, FP32)
    leaves = (hidden.requires_grad_(True), weight.requires_grad_(True))
    grads = torch.autograd.grad(layers.linear_cross_entropy(*leaves, targets), leaves)
    wide = [t.detach().double().requires_grad_(True) for t in leaves]

    def definition(h, w):
        return torch.nn.functional.cross_entropy(h @ w.T, targets)

    exact = torch.autograd.grad(definition(*wide), wide)
    step = 0.02
    length = sum(float(x.double().square().sum()) for x in grads)**0.5
    along = [x.double() / length for x in grads]
    derivative = sum(float((a * e).sum()) for a, e in zip(along, exact))

    def slope(loss, h, w):
        with torch.no_grad():
            up, down = (loss(h + s * step * along[0].to(h.dtype), w + s * step * along[1].to(w.dtype)).double() for s in (1.0, -1.0))
        return float(up - down) / (2 * step)

    left_out = abs(slope(definition, *wide) - derivative)
    # moved FP32 inputs are rounded: 2^-24 of |h| and |w| along the gradient, below 1e-6 in the loss
    difference = slope(lambda h, w: layers.linear_cross_entropy(h, w, targets), hidden.detach(), weight.detach())
    assert abs(difference - length) <= left_out + (1e-5 + 1e-6) / step


# ------------------------------------------------------------ autograd's other ways

def _each_layer(leaf):
    """The three layers as functions of one leaf [4, 64]."""
    tokens = torch.tensor([[0, 3, 1, 1]], device="cuda")
    yield lambda: layers.layer_norm(leaf)
    yield lambda: layers.embedding(tokens, leaf)
    yield lambda: layers.linear_cross_entropy(leaf, leaf.detach().clone(), tokens[0])


def test_differentiating_the_gradients_again_is_refused():
    leaf = _randn(_generator(131), 4, 64).requires_grad_(True)
    for call in _each_layer(leaf):
        (grad,) = torch.autograd.grad(call().sum(), leaf, create_graph=True)
        (plain,) = torch.autograd.grad(call().sum(), leaf)
        assert torch.equal(grad.detach(), plain)
        with pytest.raises(RuntimeError, match="first-order"):
            grad.square().sum().backward()


def test_inference_mode_and_recomputation():
    from torch.utils.checkpoint import checkpoint

    leaf = _randn(_generator(137), 4, 64).requires_grad_(True)
    for call in _each_layer(leaf):
        out = call()
        with torch.inference_mode():
            assert torch.equal(call(), out)
        (expected,) = torch.autograd.grad(out.sum(), leaf, retain_graph=True)
        (again,) = torch.autograd.grad(out.sum(), leaf)
        (recomputed,) = torch.autograd.grad(checkpoint(call, use_reentrant=False).sum(), leaf)
        assert torch.equal(again, expected) and torch.equal(recomputed, expected)


def test_inputs_changed_before_the_backward_are_refused():
    weight = _randn(_generator(139), 64).requires_grad_(True)
    x = _randn(_generator(140), 4, 64)
    out = layers.layer_norm(x, weight)
    x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


# ----------------------------------------------------------- streams, capture

def _training_pass(tokens, table, positions, weight, bias, head, targets):
    x = layers.embedding(tokens, table, positions, dtype=BF16)
    y = layers.layer_norm(x, weight, bias)
    loss = layers.linear_cross_entropy(y, head, targets)
    return (loss, *torch.autograd.grad(loss, (table, positions, weight, bias, head)))


def _pass_inputs(seed):
    g = _generator(seed)
    return (torch.randint(500, (2, 96), generator=g, device="cuda"), _randn(g, 500, 200).requires_grad_(True),
            _randn(g, 100, 200).requires_grad_(True), (1 + _randn(g, 200)).requires_grad_(True), _randn(g, 200).requires_grad_(True),
            (0.1 * _randn(g, 500, 200)).to(BF16).requires_grad_(True),
            torch.randint(500, (2, 96), generator=g, device="cuda").masked_fill(torch.rand(2, 96, generator=g, device="cuda") < 0.2, -100))


def test_layers_on_another_stream():
    inputs = _pass_inputs(83)
    expected = [t.detach() for t in _training_pass(*inputs)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        leaves = [t.detach().clone().requires_grad_(t.requires_grad) for t in inputs]
        got = [t.detach() for t in _training_pass(*leaves)]
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(got, expected):
        assert torch.equal(a, b)


def test_layers_captured_and_replayed():
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        static = _pass_inputs(89)
        for _ in range(2):
            _training_pass(*static)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outputs = _training_pass(*static)
    for seed in (97, 101, 103, 107):
        fresh = _pass_inputs(seed)
        with torch.no_grad():
            for to, of in zip(static, fresh):
                to.copy_(of)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in outputs]
        for a, b in zip(got, _training_pass(*fresh)):
            assert torch.equal(a, b.detach())
        torch.cuda.synchronize()


def test_layers_on_two_streams_at_once():
    """Calls that overlap share nothing: several passes on each of two streams, none waiting for the other."""
    each = [_pass_inputs(seed) for seed in (151, 157)]
    expected = [[t.detach().clone() for t in _training_pass(*inputs)] for inputs in each]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    leaves = []
    for stream, inputs in zip(streams, each):
        with torch.cuda.stream(stream):
            leaves.append([t.detach().clone().requires_grad_(t.requires_grad) for t in inputs])
    got = [[], []]
    for _ in range(4):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append([t.detach() for t in _training_pass(*leaves[k])])
    torch.cuda.synchronize()
    for results, wanted in zip(got, expected):
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, wanted))


def test_two_graphs_replayed_at_once():
    streams, graphs, outputs, expected = [], [], [], []
    for seed in (163, 167):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            static = _pass_inputs(seed)
            for _ in range(2):
                first = [t.detach().clone() for t in _training_pass(*static)]
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outputs.append(_training_pass(*static))
        streams.append(stream), graphs.append((graph, static)), expected.append(first)
    for _ in range(3):
        for stream, (graph, _static) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, wanted in zip(outputs, expected):
            assert all(torch.equal(a.detach(), b) for a, b in zip(got, wanted))


def test_layers_compiled_match_eager():
    inputs = _pass_inputs(109)
    expected = [t.detach() for t in _training_pass(*inputs)]

    def forward(tokens, table, positions, weight, bias, head, targets):
        y = layers.layer_norm(layers.embedding(tokens, table, positions, dtype=BF16), weight, bias)
        return layers.linear_cross_entropy(y, head, targets)

    compiled = torch.compile(forward, fullgraph=True, backend="aot_eager")
    loss = compiled(*inputs)
    got = (loss.detach(), *torch.autograd.grad(loss, inputs[1:6]))
    for a, b in zip(got, expected):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(compiled(*inputs), expected[0])


def test_layers_around_a_read():
    """Embedding, reads of the residual stream, norm and loss in one pass, against FP64 layers around
    the same reads: the read's output is the same, so the layers' bounds hold from it on."""
    from attnres import SourceBank

    inputs = _pass_inputs(113)
    tokens, table, positions, weight, bias, head, targets = inputs
    g = _generator(127)
    queries = [(0.1 * _randn(g, 200)).to(BF16).requires_grad_(True) for _ in range(2)]
    x = layers.embedding(tokens, table, positions, dtype=BF16)
    bank = SourceBank(3)
    bank.push(x)
    bank.push(layers.layer_norm(x, weight, bias))
    read = bank.read(queries[0])
    bank.push(layers.layer_norm(read, weight, bias))
    last = bank.read(queries[1])
    last.retain_grad()
    loss = layers.linear_cross_entropy(last, head, targets)
    loss.backward()
    with torch.no_grad():
        values, bounds = reference.loss(last, head, targets, -100, "mean", torch.ones((), device="cuda"))
    for name, actual, value, bound in zip(("loss", "dH", "dW"), (loss.detach(), last.grad, head.grad), values, bounds):
        assert_within(name, actual, value, bound)
    for leaf in (table, positions, weight, bias, *queries):
        assert leaf.grad is not None and bool(leaf.grad.isfinite().all()) and bool(leaf.grad.any())
