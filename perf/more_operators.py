"""Timed cases of the gated feed-forward block and of the AdamW step over many tensors.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare` holds
what a program has before a call and `run` is the call: the package's
(`attnres.layers`, `attnres.optim`) where `own` is true, else the same operator in
elementary torch operations in FP32.  `exact` is the operator's definition in FP64.

* ``ffn``:   ``(act(x @ gate.T) * (x @ up.T)) @ down.T`` of rows ``[N, D]`` with ``gate``
  and ``up`` as one weight ``[2F, D]`` and ``down`` ``[D, F]``; ``train`` adds the
  gradients of the rows and of both weights.  Rows are a layer norm's output: a
  standard deviation of about 1, 1% of channels four times larger.
* ``adamw``: one step over all tensors of a model, in place.  Parameters, gradients
  and moments are views of flat buffers, each tensor at a multiple of 256 elements (as
  sharded training keeps them), so the outputs are those buffers.  With 8-bit states a
  moment is E4M3 numbers and an FP32 scale per 256 of them, and the second moment is
  held by its root.  16-bit parameters have FP32 masters.
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
_FFN_PRODUCTS = 16384 * 4096 * 11264      # of the largest listed case, as the next
_ADAMW_ELEMENTS = 375_000_000
_BLOCK = 256                              # elements per scale of 8-bit states
_LARGEST = 448.0                          # E4M3's largest number
_LEAST = 2.0**-9                          # and its least above zero
_BETAS, _EPS, _LR, _DECAY = (0.9, 0.95), 1e-8, 3e-4, 0.1


def _ffn(rows: int, width: int, hidden: int, dtype: str, activation: str, train: bool, **name) -> dict:
    return {**name, "kind": "ffn", "rows": rows, "width": width, "hidden": hidden, "dtype": dtype,
            "activation": activation, "train": train}


def _adamw(layers: int, width: int, hidden: int, vocab: int, length: int, dtype: str, bits: int, *, step: int,
           clip: bool, **name) -> dict:
    return {**name, "kind": "adamw", "layers": layers, "width": width, "hidden": hidden, "vocab": vocab,
            "length": length, "dtype": dtype, "bits": bits, "step": step, "clip": clip}


def listed() -> list[dict]:
    return [
        # one decoded token of the 24-layer model: the shortest call
        _ffn(1, 1024, 2816, "bf16", "silu", False, name="ffn-one-token"),
        # a decoding step of 48 sequences in a wider model
        _ffn(48, 2048, 5632, "bf16", "silu", False, name="ffn-decode-48"),
        # a prompt, no gradients
        _ffn(4096, 2048, 8192, "fp16", "gelu", False, name="ffn-prompt-4k"),
        # 24-layer training workload, 2 x 1024 tokens
        _ffn(2048, 1024, 2816, "bf16", "silu", True, name="ffn-train-2k-tokens"),
        # odd sizes: rows that no wide load is aligned to
        _ffn(4095, 1537, 2051, "fp16", "gelu", True, name="ffn-train-ragged"),
        # the 24-layer model without autocast: 16 x 1024 tokens, FP32 throughout
        _ffn(16384, 1024, 2816, "fp32", "silu", True, name="ffn-train-fp32"),
        # the widest stream of the read sweep in a long batch: the largest
        _ffn(16384, 4096, 11264, "bf16", "silu", True, name="ffn-train-large"),
        # the small model of the tests and defaults: little but launches
        _adamw(2, 128, 384, 512, 64, "fp32", 32, step=3, clip=False, name="adamw-small-model"),
        # the 24-layer model in FP32
        _adamw(24, 1024, 2816, 32768, 1024, "fp32", 32, step=1000, clip=False, name="adamw-24-layers"),
        # the same with 8-bit states, gradients scaled as by clipping their norm
        _adamw(24, 1024, 2816, 32768, 1024, "fp32", 8, step=1000, clip=True, name="adamw-24-layers-8-bit"),
        # BF16 weights with FP32 masters, odd sizes
        _adamw(8, 1537, 2051, 32003, 1000, "bf16", 32, step=20000, clip=True, name="adamw-masters-ragged"),
    ]


def _log_uniform(rng: random.Random, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _round_down(rng: random.Random, value: int, low: int) -> int:
    step = rng.choice((256, 256, 64, 8, 1))  # most sizes are round, some are not
    return max(low, value // step * step)


def draw(rng: random.Random) -> dict:
    if rng.random() < 0.6:
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        width = _round_down(rng, _log_uniform(rng, 64, 4096), 64)
        hidden = _round_down(rng, _log_uniform(rng, 128, 11264), 64)
        products = _FFN_PRODUCTS // (8 if dtype == "fp32" else 2)
        rows = min(_log_uniform(rng, 1, 32768), products // (width * hidden))
        return _ffn(rows, width, hidden, dtype, rng.choice(("silu", "silu", "gelu")), rng.random() < 0.6)
    bits = rng.choice((32, 8))
    width = _round_down(rng, _log_uniform(rng, 64, 2048), 64)
    case = _adamw(rng.randint(1, 32), width, _round_down(rng, width * rng.choice((2, 3, 4)), 64),
                  _log_uniform(rng, 256, 65536), _log_uniform(rng, 16, 4096), rng.choice(("fp32", "fp32", "bf16", "fp16")),
                  bits, step=_log_uniform(rng, 1, 100000), clip=rng.random() < 0.5)
    while _elements(case) > _ADAMW_ELEMENTS // 2:
        case["layers"], case["vocab"] = max(1, case["layers"] // 2), max(256, case["vocab"] // 2)
    return case


def _sizes(case: dict) -> list[int]:
    """Elements of each parameter of the model: the tables, then per layer the norms, the
    attention's and the feed-forward's weights and the reads' queries, then the head."""
    width, hidden = case["width"], case["hidden"]
    layer = [width, width, 3 * width * width, width * width, width, width, 2 * hidden * width, width * hidden, width, width]
    return [case["vocab"] * width, case["length"] * width, *(layer * case["layers"]), case["vocab"] * width]


def _elements(case: dict) -> int:
    return sum(_sizes(case))


# ------------------------------------------------------------------- inputs

def _to_8_bits(values: torch.Tensor, least: float) -> tuple[torch.Tensor, torch.Tensor]:
    """E4M3 numbers and a scale per block; `least`: the smallest number for a value above zero."""
    blocks = values.view(-1, _BLOCK)
    scale = blocks.abs().amax(-1, keepdim=True) / _LARGEST
    numbers = blocks * torch.where(scale > 0, 1.0 / scale, 0.0)
    if least:
        numbers = torch.where(blocks > 0, numbers.clamp_min(least), numbers)
    return numbers.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def prepare(case: dict, seed: int) -> dict:
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=generator, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=generator, device="cuda")

    state = {"case": case}
    if case["kind"] == "ffn":
        rows, width, hidden, train = case["rows"], case["width"], case["hidden"], case["train"]
        channel = torch.where(rand(width) < 0.01, 4.0, 1.0)
        state["x"] = (randn(rows, width) * channel).to(dtype).requires_grad_(train)
        state["gate_up"] = randn(2 * hidden, width).mul_(width**-0.5).to(dtype).requires_grad_(train)
        state["down"] = randn(width, hidden).mul_(hidden**-0.5).to(dtype).requires_grad_(train)
        if train:  # a few tokens carry most of the gradient
            state["grad"] = (randn(rows, width) * torch.exp(1.5 * randn(rows, 1))).to(dtype)
        return state
    sizes = _sizes(case)
    first = [0]
    for size in sizes:
        first.append(first[-1] + -(-size // _BLOCK) * _BLOCK)
    total = first[-1]

    def flat(kind=torch.float32):
        return torch.zeros(total, device="cuda", dtype=kind)

    weight, grad, mean, root = flat(), flat(), flat(), flat()
    for at, size in zip(first, sizes):  # gradients of one tensor are of one magnitude, its elements' roots spread
        part = slice(at, at + size)
        magnitude = 1e-3 * torch.exp(1.5 * randn(1))
        spread = magnitude * torch.exp(randn(size))
        weight[part] = 0.02 * randn(size)
        grad[part] = spread * randn(size)
        mean[part] = 0.3 * spread * randn(size)
        root[part] = spread * (0.5 + rand(size))
    grad = grad.to(dtype)
    if case["dtype"] != "fp32":
        state["masters"] = weight
        weight = weight.to(dtype)
    state["params"], state["grads"] = weight, grad
    if case["bits"] == 8:
        state["exp_avgs"], state["exp_avg_scales"] = _to_8_bits(mean, 0.0)
        state["exp_avg_sqs"], state["exp_avg_sq_scales"] = _to_8_bits(root, _LEAST)
    else:
        state["exp_avgs"], state["exp_avg_sqs"] = mean, root.square_()
    state["grad_scale"] = 0.25 + rand(()) if case["clip"] else None

    def views(name):
        if name not in state:
            return None
        if name.endswith("scales"):
            return [state[name][a // _BLOCK:b // _BLOCK] for a, b in zip(first, first[1:])]
        return [state[name][a:a + size] for a, size in zip(first, sizes)]

    state["views"] = {name: views(name) for name in ("params", "grads", "exp_avgs", "exp_avg_sqs", "masters",
                                                     "exp_avg_scales", "exp_avg_sq_scales")}
    return state


# ---------------------------------------------------------------- the calls

_UPDATED = ("params", "exp_avgs", "exp_avg_sqs", "masters", "exp_avg_scales", "exp_avg_sq_scales")


def _run_own(state: dict):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    case = state["case"]
    if case["kind"] == "ffn":
        from attnres import layers

        leaves = (state["x"], state["gate_up"], state["down"])
        out = layers.gated_feed_forward(*leaves, activation=case["activation"])
        if not case["train"]:
            return (out,)
        return (out.detach(), *torch.autograd.grad(out, leaves, state["grad"]))
    from attnres import optim

    views = state["views"]
    optim.adamw_step(views["params"], views["grads"], views["exp_avgs"], views["exp_avg_sqs"], step=case["step"], lr=_LR,
                     betas=_BETAS, eps=_EPS, weight_decay=_DECAY, exp_avg_scales=views["exp_avg_scales"],
                     exp_avg_sq_scales=views["exp_avg_sq_scales"], masters=views["masters"], grad_scale=state["grad_scale"])
    return tuple(state[k] for k in _UPDATED if k in state)


def _plain_ffn(state: dict):
    case = state["case"]
    x, gate_up, down = (state[k].detach().float() for k in ("x", "gate_up", "down"))
    gate, up = x @ gate_up[:case["hidden"]].T, x @ gate_up[case["hidden"]:].T
    if case["activation"] == "silu":
        share = 1.0 / (1.0 + torch.exp(-gate))
    else:
        share = 0.5 * (1.0 + torch.erf(gate * 0.5**0.5))
    activated = gate * share
    product = activated * up
    dtype = state["x"].dtype
    out = (product @ down.T).to(dtype)
    if not case["train"]:
        return (out,)
    grad = state["grad"].float()
    grad_down = (grad.T @ product).to(dtype)
    grad_product = grad @ down
    if case["activation"] == "silu":
        slope = share * (1.0 + gate * (1.0 - share))
    else:
        slope = share + gate * torch.exp(-0.5 * gate * gate) * (2.0 * math.pi)**-0.5
    both = torch.cat((grad_product * up * slope, grad_product * activated), 1)
    return out, (both @ gate_up).to(dtype), (both.T @ x).to(dtype), grad_down


def _plain_adamw(state: dict):
    case = state["case"]
    weight = state.get("masters", state["params"])
    grad = state["grads"].float()
    if state["grad_scale"] is not None:
        grad = grad * state["grad_scale"]
    eighth = case["bits"] == 8
    if eighth:
        mean = (state["exp_avgs"].float().view(-1, _BLOCK) * state["exp_avg_scales"][:, None]).view(-1)
        root = (state["exp_avg_sqs"].float().view(-1, _BLOCK) * state["exp_avg_sq_scales"][:, None]).view(-1)
        square = root * root
    else:
        mean, square = state["exp_avgs"], state["exp_avg_sqs"]
    beta1, beta2 = _BETAS
    mean = mean * beta1 + grad * (1.0 - beta1)
    square = square * beta2 + grad * (1.0 - beta2) * grad
    root = torch.sqrt(square)
    move = mean / (root / math.sqrt(1.0 - beta2**case["step"]) + _EPS)
    weight.copy_(weight * (1.0 - _LR * _DECAY) - move * (_LR / (1.0 - beta1**case["step"])))
    if weight is not state["params"]:
        state["params"].copy_(weight)
    if eighth:
        for name, values, least in (("exp_avg", mean, 0.0), ("exp_avg_sq", root, _LEAST)):
            numbers, scales = _to_8_bits(values, least)
            state[name + "s"].copy_(numbers)
            state[name + "_scales"].copy_(scales)
    else:
        state["exp_avgs"].copy_(mean)
        state["exp_avg_sqs"].copy_(square)
    return tuple(state[k] for k in _UPDATED if k in state)


def run(state: dict):
    """One pass: the output, and in training the gradients; of a step, what it has updated."""
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_ffn(state) if state["case"]["kind"] == "ffn" else _plain_adamw(state)


# ---------------------------------------------------------------- the measure

def work(case: dict) -> dict:
    """Bytes of the inputs read once and the outputs written once, and the operations of
    the definition (its three products, and in training the two gradients of each)."""
    size = _BYTES[case["dtype"]]
    if case["kind"] == "ffn":
        rows, width, hidden = case["rows"], case["width"], case["hidden"]
        inputs = rows * width + 3 * width * hidden
        moved = inputs + rows * width + (inputs + rows * width if case["train"] else 0)
        return {"bytes": moved * size, "flops": 6 * rows * width * hidden * (3 if case["train"] else 1)}
    moved = 3 * size + (8 if size == 2 else 0) + (4 + 16 / _BLOCK if case["bits"] == 8 else 16)
    return {"bytes": int(_elements(case) * moved), "flops": 16 * _elements(case)}


def exact(case: dict, seed: int):
    """The definitions in FP64; the block's gradients by autograd."""
    state = prepare(case, seed)
    if case["kind"] == "ffn":
        leaves = tuple(state[k].detach().double().requires_grad_(case["train"]) for k in ("x", "gate_up", "down"))
        act = torch.nn.functional.silu if case["activation"] == "silu" else torch.nn.functional.gelu
        gate, up = torch.nn.functional.linear(leaves[0], leaves[1]).chunk(2, -1)
        out = torch.nn.functional.linear(act(gate) * up, leaves[2])
        if not case["train"]:
            return (out,)
        return (out.detach(), *torch.autograd.grad(out, leaves, state["grad"].double()))
    weight, grad = state.get("masters", state["params"]).double(), state["grads"].double()
    mean, square = state["exp_avgs"].double(), state["exp_avg_sqs"].double()
    if case["bits"] == 8:
        mean *= state["exp_avg_scales"].double().repeat_interleave(_BLOCK)
        square = (square * state["exp_avg_sq_scales"].double().repeat_interleave(_BLOCK)).square_()
    if case["clip"]:
        grad *= state["grad_scale"].double()
    mean.lerp_(grad, 1.0 - _BETAS[0])
    square.lerp_(grad.square_(), 1.0 - _BETAS[1])
    corrected = mean / (1.0 - _BETAS[0]**case["step"]), square / (1.0 - _BETAS[1]**case["step"])
    weight -= _LR * _DECAY * weight
    weight -= _LR * corrected[0] / (corrected[1].sqrt() + _EPS)
    if case["bits"] == 32:
        return (weight, mean, square) if case["dtype"] == "fp32" else (weight, mean, square, weight)
    held = []
    for values, rising in ((mean, False), (square.sqrt_(), True)):
        blocks = values.reshape(-1, _BLOCK)
        scale = blocks.abs().max(-1).values / _LARGEST
        numbers = blocks / torch.where(scale == 0, 1.0, scale)[:, None]
        if rising:
            numbers = torch.where(numbers > 0, numbers.clamp(min=_LEAST), 0.0)
        held.append((numbers.to(torch.float8_e4m3fn).double().reshape(-1), scale))
    masters = () if case["dtype"] == "fp32" else (weight,)
    return (weight, held[0][0], held[1][0], *masters, held[0][1], held[1][1])
