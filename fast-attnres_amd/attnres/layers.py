"""The layers around the residual reads, as gfx950 kernels: layer norm, embedding,
the gated feed-forward block and the softmax cross entropy of a projection to a
vocabulary.

    from attnres.layers import embedding, gated_feed_forward, layer_norm, linear_cross_entropy

They are the rest of a model's path from tokens to its loss but for its attention:
every sublayer normalises the output of a read, every other one is a feed-forward
block, the bottom looks tokens up, and the top turns the last read into a loss.  No counterpart in the reference, whose model takes
them from PyTorch (`benchmarks/model.py:180-355`).

Sums, statistics and norms are FP32; results are rounded once.  First-order
reverse-mode gradients (differentiating them again raises, and so do inputs with a
forward-mode tangent); every result and gradient is the same bits from call to call (no
floating-point atomics).  In eager mode the calls go through C++ autograd nodes
(`csrc/attnres_layers_autograd.cpp`), under ``torch.compile`` through the
``attnres_hip::`` ops below, which launch the same kernels.  Nothing
synchronises, so calls can be captured into a HIP graph.  Without the built
library every call raises.
"""

from __future__ import annotations

from typing import Any

import torch
from torch import Tensor

from . import _native
from ._ops import _OP_TAGS, _eager
from ._sources import _MAX_WIDTH, check_scalar

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_INTEGERS = (torch.int64, torch.int32)
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_MAX_TABLE = 2**30   # rows of an embedding table
_MAX_VOCAB = 2**24   # rows of a projection to a vocabulary
_MAX_TOKENS = 2**24  # of one loss
_LOSS_TILE, _MAX_TILES = 256, 2**22  # of tokens by words
_MAX_KEPT = 2**33  # bytes of exponentials
_MAX_LOOKUPS = 2**29
_MAX_PLACES = 2**26  # rows of positions
_MAX_HIDDEN = 2**16  # of a feed-forward block
_ACTIVATIONS = {"silu": 0, "gelu": 1}


# ------------------------------------------------------------------- checks

def _check_tensor(value: Any, name: str, dtypes: tuple) -> None:
    if not isinstance(value, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if value.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {', '.join(str(d).removeprefix('torch.') for d in dtypes)}")


def _check_width(width: int) -> None:
    if not 1 <= width <= _MAX_WIDTH:
        raise ValueError(f"supported envelope is 1<=D<={_MAX_WIDTH}")


def _check_place(name: str, value: Tensor, what: str, other: Tensor) -> None:
    if value.device != other.device:
        raise TypeError(f"{name} must be on the {what} device")


def _check_gpu(name: str, tensor: Tensor) -> None:
    if not tensor.is_cuda:
        raise RuntimeError(f"{name} requires CUDA (ROCm/HIP) device tensors")


def _needs_grad(*tensors: Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# --------------------------------------------------------------- layer norm

def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, *, eps: float = 1e-5) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis.

    ``x`` is ``[..., D]`` in BF16, FP16 or FP32, ``1 <= D <= 8192``; ``weight``
    and ``bias`` are ``[D]`` in ``x``'s dtype or FP32 (one dtype for both), ones
    and zeros where not given.  The result has ``x``'s shape and dtype and is
    contiguous.  ``x``'s rows may lie apart (a slice of wider rows); other
    layouts are copied.  Gradients flow to all three.
    """
    _check_tensor(x, "x", _FLOATS)
    if x.ndim < 1:
        raise ValueError("expected x [...,D]")
    _check_width(x.shape[-1])
    for name, value in (("weight", weight), ("bias", bias)):
        if value is None:
            continue
        _check_tensor(value, name, _FLOATS)
        if tuple(value.shape) != (x.shape[-1],):
            raise ValueError(f"{name} must have shape [D]")
        if value.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must have the dtype of x or FP32")
        _check_place(name, value, "x", x)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one dtype")
    eps = check_scalar(eps, "eps", positive=True)
    _check_gpu("layer_norm", x)
    if _eager(*(t for t in (x, weight, bias) if t is not None)):
        return _native.load_autograd().layer_norm(x, weight, bias, eps)
    if not _needs_grad(x, weight, bias):
        return _layer_norm_out(x, weight, bias, eps)
    return _layer_norm(x, weight, bias, eps)[0]


@torch.library.custom_op("attnres_hip::layer_norm_out", mutates_args=(), device_types="cuda", tags=_OP_TAGS)
def _layer_norm_out(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float) -> Tensor:
    return _native.load_autograd().layer_norm_forward(x, weight, bias, eps, False)[0]


@_layer_norm_out.register_fake
def _(x, weight, bias, eps):
    return x.new_empty(x.shape)


@torch.library.custom_op("attnres_hip::layer_norm", mutates_args=(), device_types="cuda", tags=_OP_TAGS)
def _layer_norm(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float) -> tuple[Tensor, Tensor]:
    return _native.load_autograd().layer_norm_forward(x, weight, bias, eps, True)


@_layer_norm.register_fake
def _(x, weight, bias, eps):
    return x.new_empty(x.shape), x.new_empty((2, x.numel() // x.shape[-1]), dtype=torch.float32)


@torch.library.custom_op("attnres_hip::layer_norm_backward", mutates_args=(), device_types="cuda", tags=_OP_TAGS)
def _layer_norm_backward(grad: Tensor, x: Tensor, weight: Tensor | None, stats: Tensor, param: torch.dtype, want_x: bool,
                         want_weight: bool, want_bias: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _native.load_autograd().layer_norm_backward(grad, x, weight, param, stats, want_x, want_weight, want_bias)


@_layer_norm_backward.register_fake
def _(grad, x, weight, stats, param, want_x, want_weight, want_bias):
    width = x.shape[-1]
    return (x.new_empty(x.shape if want_x else (0,)), x.new_empty((width if want_weight else 0,), dtype=param),
            x.new_empty((width if want_bias else 0,), dtype=param))


def _layer_norm_context(ctx: Any, inputs: tuple, output: tuple) -> None:
    x, weight, bias, _eps = inputs
    stats = output[1]
    ctx.mark_non_differentiable(stats)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, weight, stats)
    ctx.param = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype


def _layer_norm_autograd(ctx: Any, grad, _stats):
    if grad is None:
        return None, None, None, None
    x, weight, stats = ctx.saved_tensors
    wanted = ctx.needs_input_grad[:3]
    grads = _layer_norm_backward(grad, x, weight, stats, ctx.param, *wanted)
    return (*(g if want else None for g, want in zip(grads, wanted)), None)


_layer_norm.register_autograd(_layer_norm_autograd, setup_context=_layer_norm_context)


# ---------------------------------------------------------------- embedding

def embedding(tokens: Tensor, weight: Tensor, positions: Tensor | None = None, *, scale: float = 1.0,
              dtype: torch.dtype | None = None) -> Tensor:
    """``scale * weight[tokens] + positions[t]``, rounded once to ``dtype``.

    ``tokens`` is ``[..., T]``, int64 or int32; ``weight`` ``[V, D]`` and
    ``positions`` ``[P, D]`` with ``P >= T`` (row ``t`` is added to every
    sequence's ``t``-th token), both BF16, FP16 or FP32, one dtype; ``dtype``
    (default: the table's) is the result's, e.g. BF16 from an FP32 table under
    autocast.  A token outside ``0..V-1`` gives a row of NaN and takes no part
    in the table's gradient (host code that must catch one checks its tokens
    before they reach the GPU).  Gradients flow to ``weight`` (every row is written, sums
    over equal tokens in FP32 in the tokens' order) and ``positions``.
    """
    _check_tensor(tokens, "tokens", _INTEGERS)
    _check_tensor(weight, "weight", _FLOATS)
    if weight.ndim != 2:
        raise ValueError("expected weight [V,D]")
    _check_width(weight.shape[1])
    if not 1 <= weight.shape[0] <= _MAX_TABLE:
        raise ValueError(f"supported envelope is 1<=V<={_MAX_TABLE}")
    if tokens.ndim < 1 or tokens.numel() > _MAX_LOOKUPS:
        raise ValueError(f"expected tokens [...,T], at most {_MAX_LOOKUPS} of them")
    if positions is not None:
        _check_tensor(positions, "positions", _FLOATS)
        if positions.ndim != 2 or positions.shape[1] != weight.shape[1] or positions.shape[0] < tokens.shape[-1]:
            raise ValueError("positions must have shape [P,D] with P at least the tokens' last axis")
        if positions.shape[0] > _MAX_PLACES:
            raise ValueError(f"supported envelope is P<={_MAX_PLACES}")
        if positions.dtype != weight.dtype:
            raise TypeError("positions must have the dtype of weight")
        _check_place("positions", positions, "weight", weight)
    dtype = weight.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise TypeError("dtype must be bfloat16, float16 or float32")
    _check_place("tokens", tokens, "weight", weight)
    scale = check_scalar(scale, "scale")
    _check_gpu("embedding", weight)
    if _eager(*(t for t in (tokens, weight, positions) if t is not None)):
        return _native.load_autograd().embedding(tokens, weight, positions, scale, dtype)
    return _embedding(weight, positions, tokens, scale, dtype)


@torch.library.custom_op("attnres_hip::embedding", mutates_args=(), device_types="cuda", tags=_OP_TAGS)
def _embedding(weight: Tensor, positions: Tensor | None, tokens: Tensor, scale: float, dtype: torch.dtype) -> Tensor:
    return _native.load_autograd().embedding_forward(tokens, weight, positions, scale, dtype)


@_embedding.register_fake
def _(weight, positions, tokens, scale, dtype):
    return weight.new_empty((*tokens.shape, weight.shape[1]), dtype=dtype)


@torch.library.custom_op("attnres_hip::embedding_backward", mutates_args=(), device_types="cuda", tags=_OP_TAGS)
def _embedding_backward(grad: Tensor, tokens: Tensor, vocab: int, position_rows: int, table: torch.dtype, scale: float,
                        want_weight: bool, want_positions: bool) -> tuple[Tensor, Tensor]:
    return _native.load_autograd().embedding_backward(grad, tokens, vocab, position_rows, table, scale, want_weight,
                                                      want_positions)


@_embedding_backward.register_fake
def _(grad, tokens, vocab, position_rows, table, scale, want_weight, want_positions):
    width = grad.shape[-1]
    return (grad.new_empty((vocab if want_weight else 0, width), dtype=table),
            grad.new_empty((position_rows if want_positions else 0, width), dtype=table))


def _embedding_context(ctx: Any, inputs: tuple, output: Tensor) -> None:
    weight, positions, tokens, scale, _dtype = inputs
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(tokens)
    ctx.vocab, ctx.table, ctx.scale = weight.shape[0], weight.dtype, scale
    ctx.position_rows = 0 if positions is None else positions.shape[0]


def _embedding_autograd(ctx: Any, grad):
    if grad is None:
        return None, None, None, None, None
    (tokens,) = ctx.saved_tensors
    wanted = ctx.needs_input_grad[:2]
    grads = _embedding_backward(grad, tokens, ctx.vocab, ctx.position_rows, ctx.table, ctx.scale, *wanted)
    return (*(g if want else None for g, want in zip(grads, wanted)), None, None, None)


_embedding.register_autograd(_embedding_autograd, setup_context=_embedding_context)


# --------------------------------------------------------------------- loss

def linear_cross_entropy(hidden: Tensor, weight: Tensor, targets: Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", recompute: bool = False) -> Tensor:
    """Softmax cross entropy of the logits ``hidden @ weight.T``, reduced where they are formed.

    ``hidden`` is ``[..., D]``, ``weight`` ``[V, D]``, both BF16, FP16 or FP32, one
    dtype, ``1 <= D <= 8192``; ``targets`` ``[...]`` int64 or int32.  The loss is
    FP32: the mean or the sum over the targets that are not ``ignore_index``, or
    with ``reduction="none"`` a value per target (0 where ignored).  The mean of
    no targets is NaN, its gradients are zero.  Ignored tokens cost nothing and
    their hidden states are not looked at.  A target that is neither
    ``ignore_index`` nor in ``0..V-1`` makes the loss and the gradients NaN.

    16-bit inputs are multiplied on the matrix cores as they are, FP32 ones as pairs of
    FP16 numbers relative to the largest magnitude of the tensor: with FP32's 24 bits for values
    down to 2^-16 of it and, as the pairs end at 2^-40, a bit less for every further
    power of two (15 bits at 2^-25); infinities count as NaN.  (Up to 64 targets FP32 inputs
    are multiplied as they are.)

    Gradients flow to ``hidden`` and ``weight``.  Upstream gradients of
    ``reduction="none"`` may lie far apart (BF16: by 2^90): a row of ``hidden``'s gradient is as
    accurate as if it were alone; what it adds to ``weight``'s is held, for FP16 and FP32, to 2^-39 of the
    largest row of ``hidden`` times its upstream gradient.  The probabilities are rounded to the type of
    16-bit inputs for the gradients' products.

    For the gradients the forward keeps the logits' exponentials (BF16 inputs: FP16
    relative to the largest of 128, 2 bytes per target and word, the target's own unrounded;
    else FP32, 4 bytes), where that is at most 8 GiB, and the operands it has packed, in every
    live graph; beyond that, or with ``recompute=True``, it keeps 20 bytes
    per target, and the backward forms them again, for one piece of the vocabulary at a
    time, which adds a third to its products.
    """
    _check_tensor(hidden, "hidden", _FLOATS)
    _check_tensor(weight, "weight", _FLOATS)
    _check_tensor(targets, "targets", _INTEGERS)
    if hidden.ndim < 1 or weight.ndim != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("expected hidden [...,D] and weight [V,D]")
    _check_width(weight.shape[1])
    if not 1 <= weight.shape[0] <= _MAX_VOCAB:
        raise ValueError(f"supported envelope is 1<=V<={_MAX_VOCAB}")
    if tuple(targets.shape) != tuple(hidden.shape[:-1]):
        raise ValueError("targets must have the shape of hidden without its last axis")
    if targets.numel() > _MAX_TOKENS:
        raise ValueError(f"supported envelope is at most {_MAX_TOKENS} targets")
    if -(-targets.numel() // _LOSS_TILE) * -(-weight.shape[0] // _LOSS_TILE) > _MAX_TILES:
        raise ValueError(f"supported envelope is at most {_MAX_TILES} tiles of {_LOSS_TILE} targets by {_LOSS_TILE} words")
    if weight.dtype != hidden.dtype:
        raise TypeError("weight must have the dtype of hidden")
    _check_place("weight", weight, "hidden", hidden)
    _check_place("targets", targets, "hidden", hidden)
    if isinstance(ignore_index, bool) or not isinstance(ignore_index, int):
        raise TypeError("ignore_index must be an integer")
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    if not isinstance(recompute, bool):
        raise TypeError("recompute must be a bool")
    _check_gpu("linear_cross_entropy", hidden)
    code = _REDUCTIONS[reduction]
    if _eager(hidden, weight, targets):
        return _native.load_autograd().linear_cross_entropy(hidden, weight, targets, ignore_index, code, not recompute)
    keep = not recompute and _needs_grad(hidden, weight)
    return _linear_cross_entropy(hidden, weight, targets, ignore_index, code, keep)[0]


def _loss_saved_bytes(rows: int, vocab: int, width: int, dtype: torch.dtype, keep: bool) -> int:
    """attnres_hip_loss_saved_bytes, for sizes that may be symbols."""
    size = 256 + 20 * rows
    if not keep or rows == 0:
        return size
    pack = dtype == torch.float32 or width % 32 != 0
    if rows <= (64 if pack else 32):
        other, powers = 0, 4 * (16 if rows <= 16 else 32 if rows <= 32 else 64) * (-(-vocab // 128) * 128)
    else:
        width = -(-width // 32) * 32
        rows, padded = (-(-n // _LOSS_TILE) * _LOSS_TILE for n in (rows, vocab))
        powers = (2 if dtype == torch.bfloat16 else 4) * rows * padded
        operands = 2 * rows * width + (-(-2 * vocab * width // 256) * 256 if pack else 0)
        other = 8 * (padded // 128) * rows + (2 if dtype == torch.float32 else 1) * operands
        if dtype == torch.bfloat16:
            other = other + 4 * rows  # the targets' logits
    return size if powers > _MAX_KEPT else -(-size // 256) * 256 + other + powers


@torch.library.custom_op("attnres_hip::linear_cross_entropy", mutates_args=(), device_types="cuda", tags=_OP_TAGS)
def _linear_cross_entropy(hidden: Tensor, weight: Tensor, targets: Tensor, ignore_index: int, reduction: int,
                          keep: bool) -> tuple[Tensor, Tensor]:
    return _native.load_autograd().loss_forward(hidden, weight, targets, ignore_index, reduction, keep)


@_linear_cross_entropy.register_fake
def _(hidden, weight, targets, ignore_index, reduction, keep):
    saved = _loss_saved_bytes(targets.numel(), weight.shape[0], weight.shape[1], weight.dtype, keep)
    return (hidden.new_empty(targets.shape if reduction == 0 else (), dtype=torch.float32),
            hidden.new_empty((saved,), dtype=torch.uint8))


@torch.library.custom_op("attnres_hip::linear_cross_entropy_backward", mutates_args=(), device_types="cuda", tags=_OP_TAGS)
def _linear_cross_entropy_backward(grad: Tensor, hidden: Tensor, weight: Tensor, saved: Tensor, reduction: int, keep: bool,
                                   want_hidden: bool, want_weight: bool) -> tuple[Tensor, Tensor]:
    return _native.load_autograd().loss_backward(grad, hidden, weight, saved, reduction, keep, want_hidden, want_weight)


@_linear_cross_entropy_backward.register_fake
def _(grad, hidden, weight, saved, reduction, keep, want_hidden, want_weight):
    return (hidden.new_empty(hidden.shape if want_hidden else (0,)), weight.new_empty(weight.shape if want_weight else (0,)))


def _loss_context(ctx: Any, inputs: tuple, output: tuple) -> None:
    hidden, weight, _targets, _ignore_index, reduction, keep = inputs
    saved = output[1]
    ctx.mark_non_differentiable(saved)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(hidden, weight, saved)
    ctx.reduction, ctx.keep = reduction, keep


def _loss_autograd(ctx: Any, grad, _saved):
    if grad is None:
        return None, None, None, None, None, None
    hidden, weight, saved = ctx.saved_tensors
    wanted = ctx.needs_input_grad[:2]
    grads = _linear_cross_entropy_backward(grad, hidden, weight, saved, ctx.reduction, ctx.keep, *wanted)
    return (*(g if want else None for g, want in zip(grads, wanted)), None, None, None, None)


_linear_cross_entropy.register_autograd(_loss_autograd, setup_context=_loss_context)


# ------------------------------------------------------- gated feed-forward

def gated_feed_forward(x: Tensor, gate_up: Tensor, down: Tensor, *, activation: str = "silu",
                       recompute: bool = False) -> Tensor:
    """``(act(x @ gate.T) * (x @ up.T)) @ down.T``: a model's gated feed-forward block.

    ``x`` is ``[..., D]``, ``gate_up`` ``[2F, D]`` (the gate's rows, then the up
    projection's), ``down`` ``[E, F]``, all BF16, FP16 or FP32, one dtype, ``1 <= D, E
    <= 8192``, ``1 <= F <= 65536``; ``activation`` is ``"silu"`` or ``"gelu"`` (by the error
    function).  The result is ``[..., E]``, contiguous, in ``x``'s dtype.

    Sums are FP32, and so are the projections that the activation is formed from.  What the
    second product multiplies, and in the backward the gradients of both projections, is
    rounded to 16-bit inputs' type; FP16's, where upstream gradients are below 1/4, times a power
    of two that keeps its 11 bits, and infinite beyond 2^17 times the largest of those (else 65504).
    FP32 inputs are multiplied in FP32, or in large calls as sums of three BF16 numbers, with
    FP32's 24 bits; infinities may count as NaN.

    Gradients flow to all three.  For them the forward keeps both projections, 6 bytes per
    row and hidden entry each pair (FP32: 8), in every live graph; with ``recompute=True``
    nothing, and the backward forms them again, which adds a third to its products.
    """
    for name, value in (("x", x), ("gate_up", gate_up), ("down", down)):
        _check_tensor(value, name, _FLOATS)
    if x.ndim < 1 or gate_up.ndim != 2 or x.shape[-1] != gate_up.shape[1]:
        raise ValueError("expected x [...,D] and gate_up [2F,D]")
    if down.ndim != 2 or gate_up.shape[0] != 2 * down.shape[1]:
        raise ValueError("expected gate_up [2F,D] and down [E,F]")
    _check_width(x.shape[-1])
    if not 1 <= down.shape[0] <= _MAX_WIDTH:
        raise ValueError(f"supported envelope is 1<=E<={_MAX_WIDTH}")
    if not 1 <= down.shape[1] <= _MAX_HIDDEN:
        raise ValueError(f"supported envelope is 1<=F<={_MAX_HIDDEN}")
    rows = x.numel() // x.shape[-1]
    if rows > _MAX_TOKENS or -(-rows // 256) * -(-down.shape[1] // 128) > _MAX_TILES:
        raise ValueError(f"supported envelope is at most {_MAX_TOKENS} rows and {_MAX_TILES} tiles of 256 rows by 128 hidden entries")
    for name, value in (("gate_up", gate_up), ("down", down)):
        if value.dtype != x.dtype:
            raise TypeError(f"{name} must have the dtype of x")
        _check_place(name, value, "x", x)
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be 'silu' or 'gelu'")
    if not isinstance(recompute, bool):
        raise TypeError("recompute must be a bool")
    _check_gpu("gated_feed_forward", x)
    code = _ACTIVATIONS[activation]
    if _eager(x, gate_up, down):
        return _native.load_autograd().gated_feed_forward(x, gate_up, down, code, not recompute)
    keep = not recompute and _needs_grad(x, gate_up, down)
    return _gated_feed_forward(x, gate_up, down, code, keep)[0]


def _feed_forward_saved_bytes(rows: int, hidden: int, dtype: torch.dtype) -> int:
    """attnres_hip_gated_ffn_saved_bytes, for sizes that may be symbols."""
    return -(-rows // 16) * (-(-hidden // 32) * 2) * (2048 if dtype == torch.float32 else 1536)


@torch.library.custom_op("attnres_hip::gated_feed_forward", mutates_args=(), device_types="cuda", tags=_OP_TAGS)
def _gated_feed_forward(x: Tensor, gate_up: Tensor, down: Tensor, activation: int, keep: bool) -> tuple[Tensor, Tensor]:
    return _native.load_autograd().feed_forward_forward(x, gate_up, down, activation, keep)


@_gated_feed_forward.register_fake
def _(x, gate_up, down, activation, keep):
    rows = x.numel() // x.shape[-1]
    saved = _feed_forward_saved_bytes(rows, down.shape[1], x.dtype) if keep else 0
    return x.new_empty((*x.shape[:-1], down.shape[0])), x.new_empty((saved,), dtype=torch.uint8)


@torch.library.custom_op("attnres_hip::gated_feed_forward_backward", mutates_args=(), device_types="cuda", tags=_OP_TAGS)
def _gated_feed_forward_backward(grad: Tensor, x: Tensor, gate_up: Tensor, down: Tensor, saved: Tensor, activation: int, want_x: bool,
                                 want_gate_up: bool, want_down: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _native.load_autograd().feed_forward_backward(grad, x, gate_up, down, saved, activation, want_x, want_gate_up, want_down)


@_gated_feed_forward_backward.register_fake
def _(grad, x, gate_up, down, saved, activation, want_x, want_gate_up, want_down):
    return (x.new_empty(x.shape if want_x else (0,)), gate_up.new_empty(gate_up.shape if want_gate_up else (0,)),
            down.new_empty(down.shape if want_down else (0,)))


def _gated_feed_forward_context(ctx: Any, inputs: tuple, output: tuple) -> None:
    x, gate_up, down, activation, _keep = inputs
    saved = output[1]
    ctx.mark_non_differentiable(saved)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, gate_up, down, saved)
    ctx.activation = activation


def _gated_feed_forward_autograd(ctx: Any, grad, _saved):
    if grad is None:
        return None, None, None, None, None
    x, gate_up, down, saved = ctx.saved_tensors
    wanted = ctx.needs_input_grad[:3]
    grads = _gated_feed_forward_backward(grad, x, gate_up, down, saved, ctx.activation, *wanted)
    return (*(g if want else None for g, want in zip(grads, wanted)), None, None)


_gated_feed_forward.register_autograd(_gated_feed_forward_autograd, setup_context=_gated_feed_forward_context)


__all__ = ["embedding", "gated_feed_forward", "layer_norm", "linear_cross_entropy"]
