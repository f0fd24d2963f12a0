"""Forward-mode derivatives: calls that cannot carry a tangent refuse it instead of dropping it."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from attnres import SharedSources, SourceBank, attnres, layers

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _randn(*shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(sum(shape)), device="cuda").to(dtype)


def _layer_calls():
    """(name, function of a dict of its tensors, the tensors that can have a tangent)."""
    tokens = torch.tensor([[0, 3, 1, 1]], device="cuda")
    return [
        ("layer_norm", lambda t: layers.layer_norm(t["x"], t["w"], t["b"]),
         {"x": _randn(4, 64), "w": _randn(64), "b": _randn(64)}),
        ("embedding", lambda t: layers.embedding(tokens, t["w"], t["p"]), {"w": _randn(5, 64), "p": _randn(4, 64)}),
        ("linear_cross_entropy", lambda t: layers.linear_cross_entropy(t["h"], t["w"], tokens[0]),
         {"h": _randn(4, 64), "w": _randn(5, 64)}),
    ]


def _read_calls():
    def bank(tensors):
        b = SourceBank(2)
        b.push(tensors["s"]), b.push(tensors["s"] * 2)
        return b.read(tensors["q"])

    rows = {"s": _randn(3, 64, dtype=BF16), "q": _randn(64, dtype=BF16)}
    return [
        ("packed", lambda t: attnres(torch.stack((t["s"], t["s"])), t["q"]), rows),
        ("list", lambda t: attnres([t["s"], t["s"]], t["q"]), rows),
        ("shared", lambda t: SharedSources([t["s"], t["s"]]).read(t["q"]), rows),
        ("bank", bank, rows),
    ]


def _check(call, tensors):
    expected = call(tensors)
    # the tangent of an upstream gradient
    leaves = {k: v.clone().requires_grad_(True) for k, v in tensors.items()}
    out = call(leaves)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward|jvp"):
        torch.autograd.grad(out, list(leaves.values()), forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))
    for name in tensors:
        for grad in (False, True):
            for enabled in (True, False):
                leaves = {k: v.clone().requires_grad_(grad) for k, v in tensors.items()}
                with forward_ad.dual_level(), torch.set_grad_enabled(enabled):
                    leaves[name] = forward_ad.make_dual(leaves[name], torch.ones_like(leaves[name]))
                    with pytest.raises(RuntimeError, match="forward|jvp"):
                        call(leaves)
    # without a tangent inside a level, and where forward mode is off, the call is the plain one
    with forward_ad.dual_level():
        assert torch.equal(call(tensors), expected)
        dual = {k: forward_ad.make_dual(v, torch.ones_like(v)) for k, v in tensors.items()}
        with torch.inference_mode():
            assert torch.equal(call({k: v.detach() for k, v in tensors.items()}), expected)
        with forward_ad._set_fwd_grad_enabled(False):
            assert torch.equal(call(dual), expected)


@pytest.mark.parametrize("index", range(3), ids=["layer_norm", "embedding", "linear_cross_entropy"])
def test_layers_refuse_tangents(index):
    _name, call, tensors = _layer_calls()[index]
    _check(call, tensors)


def _check_compiled(call, tensors):
    compiled = torch.compile(call, fullgraph=True, backend="aot_eager")
    expected = call(tensors)
    for name in tensors:
        with forward_ad.dual_level():
            leaves = {**tensors, name: forward_ad.make_dual(tensors[name], torch.ones_like(tensors[name]))}
            with pytest.raises(RuntimeError, match="forward|jvp"):
                compiled(leaves)
    assert torch.equal(compiled(tensors), expected)


@pytest.mark.parametrize("index", range(3), ids=["layer_norm", "embedding", "linear_cross_entropy"])
def test_compiled_layers_refuse_tangents(index):
    _check_compiled(*_layer_calls()[index][1:])


@pytest.mark.parametrize("index", range(4), ids=["packed", "list", "shared", "bank"])
def test_reads_refuse_tangents(index):
    _name, call, tensors = _read_calls()[index]
    _check(call, tensors)


@pytest.mark.parametrize("index", range(2), ids=["packed", "list"])
def test_compiled_reads_refuse_tangents(index):
    _check_compiled(*_read_calls()[index][1:])
