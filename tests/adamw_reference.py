"""FP64 definition of the AdamW step, and how far FP32 arithmetic may be off.

Bounds are elementwise: `K` units of 2^-24 for each of the values that the step adds up or divides, with K = 8 covering the
roundings in a row on the way to one (the factors' own, products, sum, root, quotient).
"""

from __future__ import annotations

import torch

from layer_reference import FLOOR, HALF_STEP, U32

BLOCK = 256
K = 8 * U32


def decoded(numbers: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What 8-bit states stand for, in FP64 (dense tensors, elements as they lie)."""
    flat = numbers.as_strided((numbers.numel(),), (1,)).double()
    values = flat * scales.double().repeat_interleave(BLOCK)[:flat.numel()]
    return torch.empty_like(numbers, dtype=torch.float64).as_strided((flat.numel(),), (1,)).copy_(values).as_strided(
        numbers.shape, numbers.stride())


def step(weight, grad, mean, square, *, step, lr, betas, eps, weight_decay, grad_scale=None):
    """((w, m, v), bounds), all FP64; `mean` and `square` (v) as FP64 or FP32 values."""
    w, g, m, v = (t.double() for t in (weight, grad, mean, square))
    if grad_scale is not None:
        g = g * grad_scale.double()
    b1, b2 = betas
    m_new, v_new = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    off_m = K * (b1 * m.abs() + (1 - b1) * g.abs()) + 2.0**-149
    off_v = K * v_new + 2.0**-147
    root, unbias = v_new.sqrt(), (1 - b2**step) ** -0.5
    off_root = torch.where(root > 0, off_v / root.clamp_min(1e-300), off_v.sqrt()).clamp_max(off_v.sqrt()) + K * root
    divisor = root * unbias + eps
    rate = lr / (1 - b1**step)
    move = rate * m_new / divisor
    w_new = w * (1 - lr * weight_decay) - move
    relative = (off_root * unbias + K * divisor) / divisor
    off_w = K * (w.abs() + move.abs()) + rate * off_m / divisor * (1 + 2 * relative) + 2 * relative * move.abs() + 2.0**-149
    return (w_new, m_new, v_new), (off_w, off_m, off_v)


def assert_rounded(name, numbers, scales, values, off, root=False):
    """8-bit states are the nearest numbers: half a step of 3 bits, or of the least numbers, of the block's scale; a
    root above zero never zero.  `off`: how far FP32 may be from `values` before the rounding."""
    flat, off = (t.as_strided((t.numel(),), (1,)) for t in (values, off))
    blocks = -(-flat.numel() // BLOCK)
    padded = torch.zeros(blocks * BLOCK, dtype=torch.float64, device=flat.device)
    padded[:flat.numel()] = flat.abs()
    most = padded.view(blocks, BLOCK).amax(1) / 448
    slack = torch.zeros_like(padded)
    slack[:flat.numel()] = off
    assert bool(((scales.double() - most).abs() <= K * most + slack.view(blocks, BLOCK).amax(1) / 448 + 2.0**-126).all()), name
    scale = scales.double().repeat_interleave(BLOCK)[:flat.numel()]
    got = numbers.as_strided((numbers.numel(),), (1,)).double()
    if root:
        assert bool((got >= 0).all()) and bool((got[(flat > off) & (scale > 0)] > 0).all()), name
    limit = torch.maximum(2.0**-4 * flat.abs(), 2.0**-10 * scale) * (1 + K) + 2 * off + 2.0**-117
    if root:
        limit = torch.where(flat < 2.0**-9 * scale, 2.0**-9 * scale + limit, limit)
    worst = ((got * scale - flat).abs() - limit).max() if flat.numel() else 0.0
    assert float(worst) <= 0.0, (name, float(worst))


__all__ = ["BLOCK", "FLOOR", "HALF_STEP", "K", "assert_rounded", "decoded", "step"]
