"""The optimizer step of a training loop, as gfx950 kernels: AdamW over all tensors of
a model in a few launches, with states in 32 or in 8 bits.

    from attnres.optim import AdamW

    optimizer = AdamW(model.parameters(), lr=3e-4, weight_decay=0.1, state_bits=8)

`adamw_step` is the step itself, over lists of tensors that the caller keeps; `AdamW`
keeps them as a ``torch.optim.Optimizer``.  No counterpart in the reference, whose training
step takes the optimizer from PyTorch (`benchmarks/model.py:504-530`).

The arithmetic is FP32 throughout.  Nothing synchronises; with the step count (and, to
change it between replays, the learning rate) on the device a step can be captured into
a HIP graph.  Without the built library every call raises.
"""

from __future__ import annotations

from typing import Any, Callable, Iterable, Iterator, Sequence

import torch
from torch import Tensor

from . import _native
from ._sources import check_scalar

BLOCK = 256             # elements per scale of 8-bit states
_LEAST_OF_8_BITS = 4096  # elements; smaller tensors keep 32-bit states


def _check_factor(value: Any, name: str) -> float:
    number = check_scalar(value, name)
    if number < 0.0:
        raise ValueError(f"{name} must not be negative")
    return number


def _check_betas(betas: Any) -> tuple[float, float]:
    if not isinstance(betas, (tuple, list)) or len(betas) != 2:
        raise TypeError("betas must be a pair")
    pair = tuple(check_scalar(beta, "betas") for beta in betas)
    if not all(0.0 <= beta < 1.0 for beta in pair):
        raise ValueError("betas must be in [0, 1)")
    return pair


def _same_order(a: Tensor, b: Tensor) -> bool:
    """Whether the elements of both, of one shape, lie in one order."""
    return a.stride() == b.stride() or (a.is_contiguous() and b.is_contiguous())


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor], *,
               step: int | Tensor, lr: float | Tensor, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, exp_avg_scales: Sequence[Tensor] | None = None,
               exp_avg_sq_scales: Sequence[Tensor] | None = None, masters: Sequence[Tensor] | None = None,
               grad_scale: Tensor | None = None) -> None:
    """One AdamW step (decoupled weight decay) over all tensors, in place::

        g = grad * grad_scale
        m = beta1 * m + (1 - beta1) * g
        v = beta2 * v + (1 - beta2) * g**2
        w = w * (1 - lr * weight_decay) - lr / (1 - beta1**step) * m / (sqrt(v / (1 - beta2**step)) + eps)

    ``params`` are BF16, FP16 or FP32, one dtype, dense (in any order of axes); ``grads`` have
    their shapes and their dtype or FP32.  Gradients in another order of elements than
    their parameters are copied.  ``step`` counts from 1; it may be an int64 tensor of one element
    on the GPU, ``lr`` an FP32 one, as a captured step needs them.  ``grad_scale`` is an FP32
    tensor of one element that multiplies every gradient (clipping, loss scaling).

    The states ``exp_avgs`` (m) and ``exp_avg_sqs`` (v) have the parameters' shapes and strides: FP32, or
    with scales ``float8_e4m3fn`` and per parameter an FP32 vector of a scale for every
    256 elements as they lie; m is number times scale, and ``exp_avg_sqs`` holds v's root in
    the same way.  They are rounded to nearest, relative to the block's largest magnitude over 448 (3 bits of
    mantissa, half of the least number at 2^-19 of the largest); a root above zero is never
    rounded to zero.  A gradient that is not finite makes its element NaN or infinite, and the
    8-bit moments of its block NaN; one whose square leaves FP32, the block's second moment.

    ``masters`` are FP32 weights of 16-bit parameters: w above, of which the parameters get the
    rounded values.  Without them 16-bit parameters are read, and the new ones rounded to nearest.

    No two of the tensors may overlap.
    """
    betas = _check_betas(betas)
    eps, weight_decay = _check_factor(eps, "eps"), _check_factor(weight_decay, "weight_decay")
    on_device = isinstance(step, Tensor)
    if not on_device:
        if isinstance(step, bool) or not isinstance(step, int):
            raise TypeError("step must be an integer or a tensor")
        if not 1 <= step < 2**63:
            raise ValueError("step must be at least 1")
    rate = 0.0 if isinstance(lr, Tensor) else _check_factor(lr, "lr")
    if grad_scale is not None and not isinstance(grad_scale, Tensor):
        raise TypeError("grad_scale must be a tensor")
    _native.load_autograd().adamw_step(
        params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, masters, rate,
        lr if isinstance(lr, Tensor) else None, *betas, eps, weight_decay, 1 if on_device else step, step if on_device else None,
        grad_scale)


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is `adamw_step`, over all parameters of a group at once.

    ``state_bits=8`` keeps the moments of parameters of at least 4096 elements in 8 bits (smaller ones in
    32); ``masters=True`` keeps FP32 weights of BF16 and FP16 parameters, made from the
    parameters at their first step, or at the first one after a state dict without them.  ``capturable=True`` keeps the step count on the
    GPU, for steps in a HIP graph (take one step before capturing); ``lr`` may be an FP32
    tensor of one element on the GPU, to change it between replays.

    State dicts keep the states' dtypes, and those of ``torch.optim.AdamW`` load as 32-bit states.  Options that this
    step does not have (``amsgrad``, ``maximize``, ``differentiable``, a decay that is not decoupled) are refused, in a state
    dict too, and so are 8-bit states whose elements lie in another order than their parameter's.
    """

    def __init__(self, params: Iterable, lr: float | Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, masters: bool = False, capturable: bool = False) -> None:
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, masters=masters,
                        capturable=capturable, fused=True)
        self._check_options(defaults)
        super().__init__(params, defaults)

    @staticmethod
    def _check_options(options: dict) -> None:
        if not isinstance(options["lr"], Tensor):
            _check_factor(options["lr"], "lr")
        _check_betas(options["betas"])
        for name in ("eps", "weight_decay"):
            _check_factor(options[name], name)
        if options["state_bits"] not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        for name in ("masters", "capturable"):
            if not isinstance(options[name], bool):
                raise TypeError(f"{name} must be a bool")
        for name in ("amsgrad", "maximize", "differentiable"):
            if options.get(name):
                raise ValueError(f"AdamW has no {name}")
        if not options.get("decoupled_weight_decay", True) and options["weight_decay"] != 0.0:
            raise ValueError("AdamW's weight decay is decoupled")

    def add_param_group(self, param_group: dict) -> None:
        """As in ``torch.optim.Optimizer``, with the group's options checked."""
        self._check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def _own_state(self, p: Tensor, group: dict, shared: dict) -> dict:
        """The parameter's state, made at its first step; `shared`: device step counts made in this call."""
        state = self.state[p]
        lacks_master = group["masters"] and p.dtype != torch.float32 and "master" not in state  # a loaded state may, too
        if state and not lacks_master:
            return state
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW's state must exist before a step is captured: take one step first")
        if not state:
            if not p.is_cuda:
                raise RuntimeError("AdamW requires CUDA (ROCm/HIP) device parameters")
            if group["capturable"]:
                if p.device not in shared:
                    shared[p.device] = torch.zeros((), dtype=torch.int64, device=p.device)
                state["step"] = shared[p.device]
            else:
                state["step"] = 0
            eighth = group["state_bits"] == 8 and p.numel() >= _LEAST_OF_8_BITS
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros_like(p, dtype=torch.float8_e4m3fn if eighth else torch.float32)
                if eighth:
                    state[name + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
        if lacks_master:
            state["master"] = p.detach().to(torch.float32, copy=True)
        return state

    @torch.no_grad()
    def step(self, closure: Callable | None = None, *, grad_scale: Tensor | None = None) -> Any:
        """One step of every parameter that has a gradient; ``grad_scale`` as in `adamw_step`."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            self._step_group(group, grad_scale)
        return loss

    def _step_group(self, group: dict, grad_scale: Tensor | None) -> None:
        capturing = any(p.is_cuda for p in group["params"]) and torch.cuda.is_current_stream_capturing()
        if capturing and not group["capturable"]:
            raise RuntimeError("AdamW must be built with capturable=True for a step that is captured")
        buckets: dict[tuple, list] = {}
        shared: dict = {}
        counts: dict[int, Tensor] = {}  # on the device, by id
        taken: set[int] = set()         # counts whose step was made; a step that is refused is not counted
        for p in group["params"]:
            if p.grad is None:
                continue
            if p.grad.is_sparse:
                raise RuntimeError("AdamW takes dense gradients")
            state = self._own_state(p, group, shared)
            count = state["step"]
            if isinstance(count, Tensor):
                counts[id(count)] = count
                key = id(count)
            else:
                key = count + 1
            buckets.setdefault((p.device, p.dtype, p.grad.dtype, state["exp_avg"].dtype, "master" in state, key), []).append((p, state))
        if counts:
            # parameters without a gradient that share a count with others keep theirs
            left: dict[int, Tensor] = {}
            for p in group["params"]:
                count = self.state[p].get("step") if p.grad is None and p in self.state else None
                if isinstance(count, Tensor) and id(count) in counts:
                    if capturing:
                        raise RuntimeError("a captured step must have the gradients of the step before it")
                    if id(count) not in left:
                        left[id(count)] = count.clone()
                    self.state[p]["step"] = left[id(count)]
            for count in counts.values():
                count.add_(1)
        try:
            for (_device, _dtype, _grad, kind, has_master, key), members in buckets.items():
                states = [state for _, state in members]
                count = counts.get(key)
                eighth = kind == torch.float8_e4m3fn
                adamw_step([p for p, _ in members], [p.grad for p, _ in members], [s["exp_avg"] for s in states],
                           [s["exp_avg_sq"] for s in states], step=key if count is None else count, lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"],
                           exp_avg_scales=[s["exp_avg_scale"] for s in states] if eighth else None,
                           exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states] if eighth else None,
                           masters=[s["master"] for s in states] if has_master else None, grad_scale=grad_scale)
                taken.add(key)
                if count is None:
                    for state in states:
                        state["step"] = key
        except Exception:
            for key, count in counts.items():
                if key not in taken:
                    count.sub_(1)
            raise

    def load_state_dict(self, state_dict: dict) -> None:
        """As in ``torch.optim.Optimizer``, hooks included, but that the states keep the dtypes they were saved in,
        and options that the saved groups do not name (those of torch's) stay as they are."""
        loaded = {}
        own = [{name: group[name] for name in self.defaults} for group in self.param_groups]

        def before(_optimizer: Any, state_dict: dict) -> None:  # after the caller's hooks, so as they leave it
            for group in state_dict["param_groups"]:
                self._check_options({**self.defaults, **group})
            self._check_state(state_dict)
            loaded.update(state_dict)

        def after(_optimizer: Any) -> None:  # before the caller's
            for group, options in zip(self.param_groups, own):
                for name, value in options.items():
                    group.setdefault(name, value)
                group["fused"] = True
            self._take_state(loaded)

        hooks = (self.register_load_state_dict_pre_hook(before), self.register_load_state_dict_post_hook(after, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _saved_states(self, state_dict: dict) -> Iterator[tuple[Tensor, dict, dict]]:
        """(parameter, its group, its saved state) of the parameters that have one."""
        saved_ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        for index, (p, group) in zip(saved_ids, [(p, group) for group in self.param_groups for p in group["params"]]):
            if state_dict["state"].get(index):
                yield p, group, state_dict["state"][index]

    def _check_state(self, state_dict: dict) -> None:
        for p, _group, saved in self._saved_states(state_dict):
            for name in ("exp_avg", "exp_avg_sq", "master"):
                value = saved.get(name)
                if value is None:
                    continue
                if value.shape != p.shape:
                    raise ValueError(f"{name} must have the shape of its parameter")
                # a scale is of 256 elements as they lie
                if value.dtype == torch.float8_e4m3fn and not _same_order(value, p):
                    raise ValueError(f"an 8-bit {name} lies in another order of elements than its parameter")

    def _take_state(self, state_dict: dict) -> None:
        """The saved states in the dtypes they were saved in, in place of those that ``torch.optim.Optimizer`` has cast."""
        shared: dict[tuple, Tensor] = {}
        for p, group, saved in self._saved_states(state_dict):
            state = self.state[p] = {}
            for name in ("exp_avg", "exp_avg_sq", "master"):
                if name in saved:
                    eighth = saved[name].dtype == torch.float8_e4m3fn
                    state[name] = torch.empty_like(p, dtype=torch.float8_e4m3fn if eighth else torch.float32).copy_(saved[name])
            for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                if name in saved:
                    state[name] = saved[name].detach().to(p.device, copy=True)
            count = int(saved["step"])
            if group["capturable"]:  # parameters of one count share a tensor, as they did
                key = (id(group), p.device, count)
                if key not in shared:
                    shared[key] = torch.full((), count, dtype=torch.int64, device=p.device)
                state["step"] = shared[key]
            else:
                state["step"] = count


__all__ = ["AdamW", "adamw_step"]
