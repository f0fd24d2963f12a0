"""The layers' public functions and C ABI on the CPU: refusals, shapes under fake
tensors, and the binding against the header.  Nothing launches."""

from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

from attnres import _native, layers
from test_native_abi import _C_TYPES

HEADER = Path(__file__).resolve().parents[1] / "include" / "attnres_layers_hip.h"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _norm(x=torch.zeros(3, 8), weight=torch.ones(8), bias=torch.zeros(8), **kw):
    return layers.layer_norm(x, weight, bias, **kw)


def _embed(tokens=torch.zeros(2, 3, dtype=torch.int64), weight=torch.zeros(5, 8), positions=torch.zeros(4, 8), **kw):
    return layers.embedding(tokens, weight, positions, **kw)


def _loss(hidden=torch.zeros(2, 3, 8), weight=torch.zeros(5, 8), targets=torch.zeros(2, 3, dtype=torch.int64), **kw):
    return layers.linear_cross_entropy(hidden, weight, targets, **kw)


@pytest.mark.parametrize("call", [_norm, _embed, _loss])
def test_cpu_tensors_are_refused_after_everything_else(call):
    with pytest.raises(RuntimeError, match="CUDA"):
        call()


@pytest.mark.parametrize("call,error,match", [
    (lambda: _norm([1.0]), TypeError, "tensor"),
    (lambda: _norm(torch.zeros(3, 8, dtype=torch.float64)), TypeError, "bfloat16"),
    (lambda: _norm(torch.zeros(())), ValueError, "expected x"),
    (lambda: _norm(torch.zeros(3, 8193), None, None), ValueError, "envelope"),
    (lambda: _norm(torch.zeros(3, 0), None, None), ValueError, "envelope"),
    (lambda: _norm(weight=torch.ones(7)), ValueError, "shape"),
    (lambda: _norm(bias=torch.ones(1, 8)), ValueError, "shape"),
    (lambda: _norm(weight=torch.ones(8, dtype=BF16)), TypeError, "dtype of x"),
    (lambda: _norm(torch.zeros(3, 8, dtype=BF16), bias=torch.ones(8, dtype=BF16)), TypeError, "one dtype"),
    (lambda: _norm(weight=torch.ones(8, device="meta")), TypeError, "device"),
    (lambda: _norm(eps=0.0), ValueError, "positive"),
    (lambda: _norm(eps=float("nan")), ValueError, "finite"),
    (lambda: _norm(eps="1e-5"), TypeError, "real"),
    (lambda: _embed(torch.zeros(2, 3)), TypeError, "int64"),
    (lambda: _embed(torch.zeros(2, 3, dtype=torch.int16)), TypeError, "int64"),
    (lambda: _embed(torch.zeros((), dtype=torch.int64)), ValueError, "tokens"),
    (lambda: _embed(weight=torch.zeros(5)), ValueError, "weight"),
    (lambda: _embed(weight=torch.zeros(5, 8193), positions=None), ValueError, "envelope"),
    (lambda: _embed(weight=torch.zeros(0, 8)), ValueError, "envelope"),
    (lambda: _embed(positions=torch.zeros(2, 8)), ValueError, "positions"),
    (lambda: _embed(positions=torch.zeros(4, 7)), ValueError, "positions"),
    (lambda: _embed(positions=torch.zeros(1, 8).expand(2**26 + 1, 8)), ValueError, "envelope"),
    (lambda: _embed(torch.zeros(1, dtype=torch.int64).expand(2**29 + 1), positions=None), ValueError, "tokens"),
    (lambda: _embed(positions=torch.zeros(4, 8, dtype=BF16)), TypeError, "dtype of weight"),
    (lambda: _embed(dtype=torch.float64), TypeError, "dtype"),
    (lambda: _embed(scale=float("inf")), ValueError, "finite"),
    (lambda: _embed(scale=True), TypeError, "real"),
    (lambda: _loss(torch.zeros(2, 3, 8, dtype=torch.float64)), TypeError, "hidden"),
    (lambda: _loss(weight=torch.zeros(5, 8, dtype=BF16)), TypeError, "dtype of hidden"),
    (lambda: _loss(weight=torch.zeros(5, 7)), ValueError, "weight"),
    (lambda: _loss(weight=torch.zeros(0, 8)), ValueError, "envelope"),
    (lambda: _loss(targets=torch.zeros(2, 3)), TypeError, "targets"),
    (lambda: _loss(targets=torch.zeros(6, dtype=torch.int64)), ValueError, "targets"),
    (lambda: _loss(targets=torch.zeros(2, 3, dtype=torch.int64, device="meta")), TypeError, "device"),
    (lambda: _loss(torch.zeros(2**22, 1, device="meta"), torch.zeros(2**16 + 1, 1, device="meta"),
                   torch.zeros(2**22, dtype=torch.int64, device="meta")), ValueError, "tiles"),
    (lambda: _loss(ignore_index=1.0), TypeError, "ignore_index"),
    (lambda: _loss(ignore_index=True), TypeError, "ignore_index"),
    (lambda: _loss(reduction="max"), ValueError, "reduction"),
    (lambda: _loss(recompute=1), TypeError, "recompute"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 3, 64, device="cuda", dtype=BF16)
        weight = torch.empty(64, device="cuda")
        out, stats = torch.ops.attnres_hip.layer_norm(x, weight, None, 1e-5)
        assert out.shape == x.shape and out.dtype == BF16 and stats.shape == (2, 6) and stats.dtype == FP32
        assert torch.ops.attnres_hip.layer_norm_out(x, None, None, 1e-5).shape == x.shape
        grads = torch.ops.attnres_hip.layer_norm_backward(x, x, weight, stats, FP32, True, True, False)
        assert [tuple(g.shape) for g in grads] == [(2, 3, 64), (64,), (0,)] and grads[1].dtype == FP32
        tokens = torch.empty(2, 3, device="cuda", dtype=torch.int64)
        table = torch.empty(10, 64, device="cuda")
        out = torch.ops.attnres_hip.embedding(table, None, tokens, 1.0, BF16)
        assert out.shape == (2, 3, 64) and out.dtype == BF16
        grads = torch.ops.attnres_hip.embedding_backward(out, tokens, 10, 0, FP32, 1.0, True, False)
        assert grads[0].shape == (10, 64) and grads[0].dtype == FP32
        head = torch.empty(10, 64, device="cuda", dtype=BF16)
        for code, shape in ((0, (2, 3)), (1, ()), (2, ())):
            loss, saved = torch.ops.attnres_hip.linear_cross_entropy(x, head, tokens, -100, code, True)
            assert loss.shape == shape and loss.dtype == FP32
        grads = torch.ops.attnres_hip.linear_cross_entropy_backward(loss, x, head, saved, 2, True, True, False)
        assert grads[0].shape == x.shape and grads[1].shape == (0,)


@pytest.mark.parametrize("rows", [0, 1, 32, 33, 64, 65, 256, 257, 32768])
@pytest.mark.parametrize("vocab,width", [(1, 64), (257, 33), (131072, 2048), (131073, 64)])
@pytest.mark.parametrize("dtype", [BF16, torch.float16, FP32])
@pytest.mark.parametrize("keep", [False, True])
def test_saved_bytes_of_the_fake_kernel(rows, vocab, width, dtype, keep):
    code = (BF16, torch.float16, FP32).index(dtype)
    expected = _native.load().attnres_hip_loss_saved_bytes(rows, vocab, width, code, keep)
    assert layers._loss_saved_bytes(rows, vocab, width, dtype, keep) == expected


# ---------------------------------------------------------------------- C ABI

def _declarations():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    found = {}
    for match in re.finditer(r"\b(?:int|int64_t)\s+(attnres_hip_\w+)\s*\(([^)]*)\)\s*;", text):
        types = []
        for param in match.group(2).split(","):
            words = " ".join(param.split())
            types.append(re.sub(r"\s*\b\w+$", "", words).replace(" *", "*"))
        found[match.group(1)] = types
    return found


def test_binding_matches_the_header():
    declared = _declarations()
    assert set(declared) == set(_native.LAYER_SIGNATURES)
    for name, types in declared.items():
        assert _native.LAYER_SIGNATURES[name][1] == [_C_TYPES[t] for t in types], name


_FAKE = 0x1000  # never dereferenced: every call below fails the host's checks


def _status(name, **overrides):
    defaults = {
        "layer_norm_forward": dict(x=_FAKE, x_stride=64, rows=3, width=64, dtype=0, weight=_FAKE, bias=_FAKE, param_dtype=2,
                                   eps=1e-5, out=_FAKE, stats=None, stream=None),
        "layer_norm_backward": dict(grad_out=_FAKE, x=_FAKE, x_stride=64, rows=3, width=64, dtype=0, weight=_FAKE, param_dtype=2,
                                    stats=_FAKE, grad_x=_FAKE, grad_weight=_FAKE, grad_bias=None, workspace=_FAKE, elems=1 << 20,
                                    stream=None),
        "embedding_forward": dict(tokens=_FAKE, token_bytes=8, batch=2, length=3, weight=_FAKE, vocab=10, width=64, weight_dtype=0,
                                  positions=None, scale=1.0, out=_FAKE, out_dtype=0, stream=None),
        "embedding_backward": dict(grad_out=_FAKE, out_dtype=0, tokens=_FAKE, token_bytes=8, batch=2, length=3, vocab=10, width=64,
                                   weight_dtype=0, scale=1.0, grad_weight=_FAKE, grad_positions=None, position_rows=0,
                                   workspace=_FAKE, bytes=1 << 30, stream=None),
        "loss_forward": dict(hidden=_FAKE, hidden_stride=64, weight=_FAKE, weight_stride=64, targets=_FAKE, target_bytes=8, rows=3,
                             vocab=10, width=64, dtype=0, ignore_index=-100, reduction=2, keep=0, loss=_FAKE, saved=_FAKE,
                             workspace=_FAKE, bytes=1 << 40, stream=None),
        "loss_backward": dict(hidden=_FAKE, hidden_stride=64, weight=_FAKE, weight_stride=64, rows=3, vocab=10, width=64, dtype=0,
                              reduction=2, keep=0, saved=_FAKE, grad_loss=_FAKE, grad_hidden=_FAKE, grad_weight=_FAKE, workspace=_FAKE,
                              bytes=1 << 40, stream=None),
    }[name]
    assert set(overrides) <= set(defaults)
    return getattr(_native.load(), f"attnres_hip_{name}")(*{**defaults, **overrides}.values())


@pytest.mark.parametrize("name,override,status", [
    ("layer_norm_forward", {"x": None}, _native.ERR_NULL_POINTER),
    ("layer_norm_forward", {"out": None}, _native.ERR_NULL_POINTER),
    ("layer_norm_forward", {"rows": -1}, _native.ERR_SHAPE),
    ("layer_norm_forward", {"width": 0}, _native.ERR_SHAPE),
    ("layer_norm_forward", {"width": 8193}, _native.ERR_SHAPE),
    ("layer_norm_forward", {"dtype": 3}, _native.ERR_SHAPE),
    ("layer_norm_forward", {"param_dtype": 1}, _native.ERR_SHAPE),
    ("layer_norm_forward", {"x_stride": -1}, _native.ERR_STRIDE),
    ("layer_norm_forward", {"eps": -1.0}, _native.ERR_SCALAR),
    ("layer_norm_forward", {"eps": float("nan")}, _native.ERR_SCALAR),
    ("layer_norm_backward", {"stats": None}, _native.ERR_NULL_POINTER),
    ("layer_norm_backward", {"elems": 2 * 64 - 1}, _native.ERR_WORKSPACE),
    ("layer_norm_backward", {"workspace": None}, _native.ERR_WORKSPACE),
    ("embedding_forward", {"tokens": None}, _native.ERR_NULL_POINTER),
    ("embedding_forward", {"token_bytes": 2}, _native.ERR_SHAPE),
    ("embedding_forward", {"vocab": 0}, _native.ERR_SHAPE),
    ("embedding_forward", {"batch": 2**20, "length": 2**20}, _native.ERR_SHAPE),
    ("embedding_forward", {"batch": 2**15 + 1, "length": 2**14}, _native.ERR_SHAPE),
    ("embedding_backward", {"grad_positions": _FAKE, "position_rows": 2**26 + 1}, _native.ERR_SHAPE),
    ("embedding_forward", {"out_dtype": 7}, _native.ERR_SHAPE),
    ("embedding_backward", {"grad_out": None}, _native.ERR_NULL_POINTER),
    ("embedding_backward", {"bytes": 100}, _native.ERR_WORKSPACE),
    ("embedding_backward", {"grad_positions": _FAKE, "position_rows": 2}, _native.ERR_SHAPE),
    ("loss_forward", {"hidden": None}, _native.ERR_NULL_POINTER),
    ("loss_forward", {"targets": None}, _native.ERR_NULL_POINTER),
    ("loss_forward", {"saved": None}, _native.ERR_NULL_POINTER),
    ("loss_forward", {"rows": 2**24 + 1}, _native.ERR_SHAPE),
    ("loss_forward", {"rows": 2**24, "vocab": 2**24}, _native.ERR_SHAPE),
    ("loss_forward", {"rows": 2**22, "vocab": 2**16 + 1}, _native.ERR_SHAPE),
    ("loss_forward", {"workspace": _FAKE + 8}, _native.ERR_WORKSPACE),
    ("loss_forward", {"saved": _FAKE + 4}, _native.ERR_WORKSPACE),
    ("loss_backward", {"workspace": _FAKE + 8}, _native.ERR_WORKSPACE),
    ("loss_forward", {"width": 8193}, _native.ERR_SHAPE),
    ("loss_forward", {"target_bytes": 1}, _native.ERR_SHAPE),
    ("loss_forward", {"reduction": 3}, _native.ERR_SCALAR),
    ("loss_forward", {"weight": _FAKE + 2}, _native.ERR_STRIDE),
    ("loss_forward", {"weight_stride": 68}, _native.ERR_STRIDE),
    ("loss_forward", {"weight_stride": 0}, _native.ERR_STRIDE),
    ("loss_forward", {"weight_stride": 2**23}, _native.ERR_STRIDE),
    ("loss_forward", {"bytes": 1000}, _native.ERR_WORKSPACE),
    ("loss_backward", {"grad_loss": None}, _native.ERR_NULL_POINTER),
    ("loss_backward", {"bytes": 1000}, _native.ERR_WORKSPACE),
    ("loss_backward", {"hidden_stride": -64}, _native.ERR_STRIDE),
])
def test_c_abi_refusals(name, override, status):
    assert _status(name, **override) == status
    assert _native.load().attnres_hip_last_error().decode()


def test_workspaces_are_of_the_shape_alone():
    lib = _native.load()
    assert lib.attnres_hip_layer_norm_workspace_elems(0, 64) == 0
    assert lib.attnres_hip_layer_norm_workspace_elems(4, 8193) == -1
    assert lib.attnres_hip_embedding_workspace_bytes(2, 3, 0, 64) == -1
    assert lib.attnres_hip_loss_workspace_bytes(3, 10, 64, 9, 0, 0) == -1
    assert lib.attnres_hip_loss_saved_bytes(-1, 10, 64, 0, 0) == -1
    # the probabilities of a large vocabulary are formed in pieces: the backward of 16384 tokens and
    # 131072 words needs far less than the 4 GiB of BF16 probabilities
    for keep in (0, 1):
        assert lib.attnres_hip_loss_workspace_bytes(16384, 131072, 2048, 0, keep, 1) < 1 << 30
    # kept exponentials: 2 bytes each and 1 / 32 of that, up to 8 GiB, and the rows that count
    assert lib.attnres_hip_loss_saved_bytes(16384, 131072, 2048, 0, 0) == 256 + 20 * 16384
    assert 1 << 32 < lib.attnres_hip_loss_saved_bytes(16384, 131072, 2048, 0, 1) < 1.04 * 2**32 + 2**26
    assert 1 << 33 < lib.attnres_hip_loss_saved_bytes(32768, 131072, 2048, 0, 1) < 1.04 * 2**33 + 2**27
    assert lib.attnres_hip_loss_saved_bytes(32769, 131072, 2048, 0, 1) == 256 + 20 * 32769
