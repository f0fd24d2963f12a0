"""Timed cases of the layers around the residual reads: layer norm, embedding and
the loss over the vocabulary.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare` holds
what a program has before a call and `run` is the call: the package's
(`attnres.layers`) where `own` is true, else the same operator in elementary torch
operations in FP32.  `exact` is the operator's definition in FP64.

* ``norm``:      layer norm of rows ``[N, D]``; ``train`` adds the gradients of the
  rows, the weight and the bias.  Rows are outputs of residual reads: a standard
  deviation of about 1, 1% of channels eight times larger, a mean per channel.
* ``embedding``: rows of a table by token, scaled, plus a row per position;
  ``train`` adds the gradients of the table and the positions.  Tokens follow a
  Zipf law, as text does.
* ``loss``:      softmax cross entropy of ``hidden @ weight.T``; ``train`` adds the
  gradients of both.  Logits have a standard deviation of about 2, and half of the
  targets a raised one, as a model in training has; a share of the targets is
  ignored (prompts, padding).
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

_PACKAGE = str(Path(__file__).resolve().parents[1] / "fast-attnres_amd")

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_IGNORE = -100
_EPS = 1e-5
_NORM_ELEMENTS = 32768 * 4096          # of the largest listed case, as the two below
_EMBEDDING_ELEMENTS = 131072 * 2048
_LOSS_PRODUCTS = 16384 * 131072 * 2048


def _norm(rows: int, width: int, dtype: str, params: str, train: bool, **name) -> dict:
    return {**name, "kind": "norm", "rows": rows, "width": width, "dtype": dtype, "params": params, "train": train}


def _embedding(batch: int, length: int, width: int, vocab: int, dtype: str, table: str, train: bool, *,
               positions: bool, scale: float, **name) -> dict:
    return {**name, "kind": "embedding", "batch": batch, "length": length, "width": width, "vocab": vocab,
            "dtype": dtype, "table": table, "train": train, "positions": positions, "scale": scale}


def _loss(rows: int, width: int, vocab: int, dtype: str, train: bool, *, reduction: str = "mean",
          ignored: float = 0.0, **name) -> dict:
    return {**name, "kind": "loss", "rows": rows, "width": width, "vocab": vocab, "dtype": dtype, "train": train,
            "reduction": reduction, "ignored": ignored}


def listed() -> list[dict]:
    return [
        # the norm after a read of one decoded token: the shortest call there is
        _norm(1, 2048, "bf16", "bf16", False, name="norm-one-token"),
        # 24-layer training workload, 2 x 1024 tokens, BF16 stream and FP32 parameters (autocast)
        _norm(2048, 1024, "bf16", "fp32", True, name="norm-train-2k-tokens"),
        # odd sizes: rows that no wide load is aligned to
        _norm(4095, 1537, "fp32", "fp32", True, name="norm-train-ragged"),
        # the widest stream of the read sweep in a long batch
        _norm(32768, 4096, "bf16", "bf16", True, name="norm-train-large"),
        # one decoding step of 16 sequences: a row each
        _embedding(16, 1, 1024, 32768, "bf16", "bf16", False, positions=False, scale=1.0, name="embedding-decode"),
        # 24-layer training workload, 2 x 1024 tokens: token and position tables in FP32, BF16 stream
        _embedding(2, 1024, 1024, 32768, "bf16", "fp32", True, positions=True, scale=1.0,
                   name="embedding-train-2k-tokens"),
        # a large vocabulary, eight long sequences, scaled by the width's root, a table in BF16
        _embedding(8, 4096, 2048, 131072, "bf16", "bf16", True, positions=False, scale=2048**0.5,
                   name="embedding-train-large-vocabulary"),
        # scoring a short continuation: a loss per token, no gradient
        _loss(16, 1024, 32768, "bf16", False, reduction="none", name="loss-score-16-tokens"),
        # 24-layer training workload, 2 x 1024 tokens
        _loss(2048, 1024, 32768, "bf16", True, name="loss-train-2k-tokens"),
        # the 24-layer model without autocast: 16 x 1024 tokens, FP32 throughout
        _loss(16384, 1024, 8192, "fp32", True, name="loss-train-fp32"),
        # instruction tuning: prompts and padding ignored, a weight per token, odd sizes
        _loss(4095, 1000, 50021, "fp16", True, reduction="none", ignored=0.35, name="loss-train-masked-ragged"),
        # long batch, large vocabulary, wide stream: the largest
        _loss(16384, 2048, 131072, "bf16", True, ignored=0.05, name="loss-train-large-vocabulary"),
    ]


def _log_uniform(rng: random.Random, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _round_down(rng: random.Random, value: int, low: int) -> int:
    step = rng.choice((256, 256, 64, 8, 1))  # most sizes are round, some are not
    return max(low, value // step * step)


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("norm", "embedding", "loss"))
    train = rng.random() < 0.75
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "norm":
        width = _round_down(rng, _log_uniform(rng, 64, 8192), 64)
        rows = min(_log_uniform(rng, 1, 65536), _NORM_ELEMENTS // width // (2 if dtype == "fp32" else 1))
        return _norm(rows, width, dtype, rng.choice((dtype, "fp32")), train)
    if kind == "embedding":
        width = _round_down(rng, _log_uniform(rng, 64, 4096), 64)
        size = 2 if dtype == "fp32" else 1
        vocab = min(_round_down(rng, _log_uniform(rng, 512, 262144), 512), _EMBEDDING_ELEMENTS // 2 // width // size)
        tokens = min(_log_uniform(rng, 1, 65536), _EMBEDDING_ELEMENTS // 8 // width // size)
        batch = min(tokens, rng.choice((1, 2, 4, rng.randint(1, 16))))
        table = dtype if rng.random() < 0.5 else "fp32"
        if table == "fp32":
            vocab = max(512, vocab // 2)
        return _embedding(batch, max(1, tokens // batch), width, vocab, dtype, table, train,
                          positions=rng.random() < 0.5, scale=rng.choice((1.0, width**0.5)))
    width = _round_down(rng, _log_uniform(rng, 128, 4096), 64)
    vocab = _round_down(rng, _log_uniform(rng, 512, 131072), 512)
    products = _LOSS_PRODUCTS // (8 if dtype == "fp32" else 2)
    rows = min(_log_uniform(rng, 1, 16384), products // (width * vocab))
    return _loss(rows, width, vocab, dtype, train, reduction=rng.choice(("mean", "mean", "sum", "none")),
                 ignored=rng.choice((0.0, 0.0, round(rng.uniform(0.0, 0.6), 2))))


# ------------------------------------------------------------------- inputs

def _ignored(case: dict) -> int:
    """How many targets are ignored; at least one stays."""
    return min(int(case["ignored"] * case["rows"]), case["rows"] - 1)


def _zipf(count: int, vocab: int, generator) -> torch.Tensor:
    """Token ids whose rank r has a probability of about 1 / r, ranks spread over the ids."""
    u = torch.rand(count, generator=generator, device="cuda", dtype=torch.float64)
    rank = torch.exp(u * math.log(vocab)).to(torch.int64).clamp_(1, vocab) - 1
    return rank * 7919 % vocab if math.gcd(7919, vocab) == 1 else rank


def prepare(case: dict, seed: int) -> dict:
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype, train = _DTYPES[case["dtype"]], case["train"]

    def randn(*shape):
        return torch.randn(*shape, generator=generator, device="cuda")

    def leaf(tensor, kind):
        return tensor.to(kind).requires_grad_(train)

    state = {"case": case}
    if case["kind"] == "norm":
        rows, width, params = case["rows"], case["width"], _DTYPES[case["params"]]
        channel = torch.where(torch.rand(width, generator=generator, device="cuda") < 0.01, 8.0, 1.0)
        state["x"] = leaf((randn(rows, width) + 0.3 * randn(width)) * channel, dtype)
        state["weight"] = leaf(1.0 + 0.2 * randn(width), params)
        state["bias"] = leaf(0.1 * randn(width), params)
        if train:
            state["grad"] = randn(rows, width).to(dtype)
    elif case["kind"] == "embedding":
        batch, length, width, vocab = case["batch"], case["length"], case["width"], case["vocab"]
        table = _DTYPES[case["table"]]
        state["tokens"] = _zipf(batch * length, vocab, generator).view(batch, length)
        state["weight"] = leaf(0.02 * randn(vocab, width), table)
        # a table of positions is longer than the sequences at hand
        state["positions"] = leaf(0.02 * randn(length + length // 4, width), table) if case["positions"] else None
        if train:
            state["grad"] = randn(batch, length, width).to(dtype)
    else:
        rows, width, vocab = case["rows"], case["width"], case["vocab"]
        weight = randn(vocab, width).mul_(2.0 / width**0.5)
        targets = _zipf(rows, vocab, generator)
        raised = 8.0 * torch.rand(rows, 1, generator=generator, device="cuda")
        state["hidden"] = leaf(randn(rows, width) + raised / 2.0 * weight[targets], dtype)
        state["weight"] = leaf(weight, dtype)
        hidden_out = torch.randperm(rows, generator=generator, device="cuda")[:_ignored(case)]
        state["targets"] = targets.index_fill(0, hidden_out, _IGNORE)
        if train:  # of the mean or the sum: one factor; per token: its weight
            upstream = torch.rand(rows if case["reduction"] == "none" else (), generator=generator, device="cuda")
            state["grad"] = upstream + 0.5
            if case["reduction"] != "mean":
                state["grad"] = state["grad"] / rows
            if case["dtype"] == "fp16":  # training in FP16 scales its loss, or its gradients vanish
                state["grad"] = state["grad"] * 1024.0
    return state


# ---------------------------------------------------------------- the calls

def _run_own(state: dict):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from attnres import layers

    case = state["case"]
    if case["kind"] == "norm":
        leaves = (state["x"], state["weight"], state["bias"])
        out = layers.layer_norm(*leaves, eps=_EPS)
    elif case["kind"] == "embedding":
        leaves = tuple(state[k] for k in ("weight", "positions") if state[k] is not None)
        out = layers.embedding(state["tokens"], *leaves, scale=case["scale"], dtype=_DTYPES[case["dtype"]])
    else:
        leaves = (state["hidden"], state["weight"])
        out = layers.linear_cross_entropy(*leaves, state["targets"], ignore_index=_IGNORE,
                                          reduction=case["reduction"])
    if not case["train"]:
        return (out,)
    return (out.detach(), *torch.autograd.grad(out, leaves, state["grad"]))


def _plain_norm(state: dict):
    x, weight, bias = (state[k].detach().float() for k in ("x", "weight", "bias"))
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + _EPS)
    hat = centred * rstd
    out = (hat * weight + bias).to(state["x"].dtype)
    if not state["case"]["train"]:
        return (out,)
    grad = state["grad"].float()
    scaled = grad * weight
    grad_x = rstd * (scaled - scaled.mean(-1, keepdim=True) - hat * (scaled * hat).mean(-1, keepdim=True))
    return (out, grad_x.to(out.dtype), (grad * hat).sum(0).to(state["weight"].dtype),
            grad.sum(0).to(state["bias"].dtype))


def _plain_embedding(state: dict):
    case, tokens, weight, positions = state["case"], state["tokens"], state["weight"], state["positions"]
    out = weight.detach()[tokens].float() * case["scale"]
    if positions is not None:
        out = out + positions.detach()[:case["length"]].float()
    out = out.to(_DTYPES[case["dtype"]])
    if not case["train"]:
        return (out,)
    grad = state["grad"].float()
    total = torch.zeros(weight.shape, device="cuda").index_add_(0, tokens.reshape(-1), grad.flatten(0, 1))
    grads = [(total * case["scale"]).to(weight.dtype)]
    if positions is not None:
        grad_positions = torch.zeros(positions.shape, device="cuda")
        grad_positions[:case["length"]] = grad.sum(0)
        grads.append(grad_positions.to(positions.dtype))
    return (out, *grads)


def _plain_loss(state: dict):
    case, targets = state["case"], state["targets"]
    hidden, weight = state["hidden"].detach().float(), state["weight"].detach().float()
    rows, vocab = case["rows"], case["vocab"]
    kept = targets != _IGNORE
    index = torch.where(kept, targets, 0)
    train = case["train"]
    if train:
        upstream = state["grad"] / kept.sum() if case["reduction"] == "mean" else state["grad"]
        upstream = torch.where(kept, upstream, 0.0)
        grad_hidden, grad_weight = torch.empty_like(hidden), torch.zeros_like(weight)
    losses = torch.empty(rows, device="cuda")
    step = max(1, 2**29 // vocab)  # logits of 2 GiB at once
    for first in range(0, rows, step):
        part = slice(first, min(rows, first + step))
        logits = hidden[part] @ weight.T
        top = logits.amax(-1, keepdim=True)
        target = logits.gather(1, index[part, None])
        logits.sub_(top).exp_()
        total = logits.sum(-1, keepdim=True)
        losses[part] = (total.log() + top - target).squeeze(1)
        if train:
            probabilities = logits.div_(total)
            probabilities.scatter_add_(1, index[part, None], torch.full_like(target, -1.0))
            probabilities.mul_(upstream[part, None])
            grad_hidden[part] = probabilities @ weight
            grad_weight += probabilities.T @ hidden[part]
    losses = torch.where(kept, losses, 0.0)
    if case["reduction"] != "none":
        losses = losses.sum()
        if case["reduction"] == "mean":
            losses = losses / kept.sum()
    if not train:
        return (losses,)
    return losses, grad_hidden.to(state["hidden"].dtype), grad_weight.to(state["weight"].dtype)


_PLAIN = {"norm": _plain_norm, "embedding": _plain_embedding, "loss": _plain_loss}


def run(state: dict):
    """One pass: the output, and in training the gradients of the inputs that have one."""
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------- the measure

def work(case: dict) -> dict:
    """Bytes of the inputs read once and the outputs written once, and the operations of
    the definition (the logits and the two gradient products; no logits twice)."""
    size, train = _BYTES[case["dtype"]], case["train"]
    if case["kind"] == "norm":
        rows, width, params = case["rows"], case["width"], _BYTES[case["params"]]
        elements = rows * width
        return {"bytes": elements * size * (4 if train else 2) + 2 * width * params * (2 if train else 1),
                "flops": elements * (19 if train else 8)}
    if case["kind"] == "embedding":
        rows, width, table = case["batch"] * case["length"], case["width"], _BYTES[case["table"]]
        read = min(rows, case["vocab"]) * width * table + 8 * rows
        extra = case["length"] * width * table if case["positions"] else 0
        moved = read + extra + rows * width * size
        if train:
            moved += rows * width * size + case["vocab"] * width * table
            if case["positions"]:
                moved += (case["length"] + case["length"] // 4) * width * table
        return {"bytes": moved, "flops": rows * width * (4 if train else 2)}
    rows, width, vocab = case["rows"], case["width"], case["vocab"]
    kept = rows - _ignored(case)
    once = (kept * width + vocab * width) * size
    return {"bytes": once + 8 * rows + ((rows * width + vocab * width) * size if train else 0),
            "flops": 2 * kept * vocab * width * (3 if train else 1)}


def exact(case: dict, seed: int):
    """The definitions in FP64, gradients by autograd; the loss's row by row block."""
    state = prepare(case, seed)

    def wide(tensor):
        return tensor.detach().double().requires_grad_(case["train"])

    if case["kind"] == "norm":
        x, weight, bias = wide(state["x"]), wide(state["weight"]), wide(state["bias"])
        out = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + _EPS).sqrt() * weight + bias
        if not case["train"]:
            return (out,)
        return (out.detach(), *torch.autograd.grad(out, (x, weight, bias), state["grad"].double()))
    if case["kind"] == "embedding":
        weight, tokens = wide(state["weight"]), state["tokens"]
        leaves = [weight]
        out = weight.index_select(0, tokens.reshape(-1)).view(*tokens.shape, -1) * case["scale"]
        if state["positions"] is not None:
            leaves.append(wide(state["positions"]))
            out = out + leaves[1].narrow(0, 0, case["length"])
        if not case["train"]:
            return (out,)
        return (out.detach(), *torch.autograd.grad(out, leaves, state["grad"].double()))
    targets = state["targets"]
    kept = (targets != _IGNORE).nonzero().squeeze(1)
    hidden, weight = state["hidden"].detach().double(), state["weight"].detach().double()
    scale = torch.ones(kept.numel(), device="cuda", dtype=torch.float64)
    if case["reduction"] == "mean":
        scale /= kept.numel()
    losses = torch.zeros(case["rows"], device="cuda", dtype=torch.float64)
    grad_hidden, grad_weight = torch.zeros_like(hidden), torch.zeros_like(weight)
    step = max(1, 2**28 // case["vocab"])
    for first in range(0, kept.numel(), step):
        at = kept[first:first + step]
        log_p = torch.log_softmax(hidden[at] @ weight.T, -1)
        chosen = torch.arange(at.numel(), device="cuda"), targets[at]
        losses[at] = -log_p[chosen]
        if case["train"]:
            upstream = scale[first:first + step]
            upstream = upstream * (state["grad"][at] if case["reduction"] == "none" else state["grad"]).double()
            term = log_p.exp_()
            term[chosen] -= 1.0
            term *= upstream[:, None]
            grad_hidden[at] = term @ weight
            grad_weight += term.T @ hidden[at]
    if case["reduction"] == "none":
        loss = losses
    else:
        loss = losses[kept].sum() / (kept.numel() if case["reduction"] == "mean" else 1)
    return (loss, grad_hidden, grad_weight) if case["train"] else (loss,)
