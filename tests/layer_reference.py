"""FP64 definitions of the layers, and how far FP32 arithmetic with one rounding may be off.

Every bound is elementwise: `u` (half a step of the output's type, relative) times the
value, plus `K * 2^-24` times the magnitudes that the FP32 arithmetic adds up, where K
counts the roundings in a row on the way to a value.
"""

from __future__ import annotations

import torch

U32 = 2.0**-24
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
# half of the smallest subnormal step: what a tiny value may lose whole
FLOOR = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}


def assert_within(name: str, actual: torch.Tensor, expected: torch.Tensor, bound: torch.Tensor | float) -> None:
    """|actual - expected| <= u |expected| + bound, NaN exactly where expected."""
    assert actual.shape == expected.shape, (name, actual.shape, expected.shape)
    got, want = actual.double(), expected.double()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), f"{name}: NaN in other places"
    limit = HALF_STEP[actual.dtype] * want.abs() + FLOOR[actual.dtype] + bound
    excess = ((got - want).abs() - limit).masked_fill(nan, -1.0)
    worst = int(excess.argmax()) if excess.numel() else 0
    assert excess.numel() == 0 or float(excess.flatten()[worst]) <= 0.0, (
        f"{name}: {float(got.flatten()[worst])} for {float(want.flatten()[worst])}, "
        f"allowed {float(limit.flatten()[worst]) if limit.dim() else float(limit)}")


def layer_norm(x, weight, bias, eps, grad):
    """(out, dx, dw, db) and the bounds of each.

    A lane adds up at most 64 elements, a tree 6 more levels and 4 wavefronts: at most
    76 roundings in a row for a mean, about 100 for an output; the deviation of x - mean
    from the mean's rounding is relative to the mean magnitude of x.  K = 256 also covers the
    columns' sums over the rows of a test (at most 16 rows in a row per lane, 32 groups, 512 partial rows of
    which a thread adds 16, then 32).
    """
    k = 256 * U32
    x, grad = x.double(), grad.double()
    width = x.shape[-1]
    w = torch.ones(width, device=x.device, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(width, device=x.device, dtype=torch.float64) if bias is None else bias.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    hat = (x - mean) * rstd
    # off-ness of hat over k: its own size, and the mean's rounding
    off = hat.abs() + rstd * x.abs().mean(-1, keepdim=True) * (1.0 + hat.abs())
    out = hat * w + b
    g = grad * w
    s1, s2 = g.mean(-1, keepdim=True), (g * hat).mean(-1, keepdim=True)
    grad_x = rstd * (g - s1 - hat * s2)
    size = g.abs() + g.abs().mean(-1, keepdim=True) + off * s2.abs() + hat.abs() * (g.abs() * off).mean(-1, keepdim=True)
    wide = 1.0 + rstd * x.abs().mean(-1, keepdim=True)  # rstd's own error

    def columns(t):
        return t.reshape(-1, width).sum(0)

    return ((out, grad_x, columns(grad * hat), columns(grad)),
            (k * (off * w.abs() + b.abs()), k * rstd * size * wide, k * columns(grad.abs() * off),
             k * columns(grad.abs())))


def embedding(tokens, weight, positions, scale, grad):
    """(out, dW, dpos) and bounds: two roundings for a row; a sum of n rows has at most
    n + 2 roundings in a row."""
    known = (tokens >= 0) & (tokens < weight.shape[0])
    index = torch.where(known, tokens, 0).long()
    out = weight.double()[index] * scale
    bound = 2 * U32 * out.abs()
    if positions is not None:
        place = positions.double()[:tokens.shape[-1]]
        bound = bound + U32 * (out.abs() + place.abs())
        out = out + place
    out = out.masked_fill(~known[..., None], float("nan"))
    grad = grad.double()
    kept = grad * known[..., None]
    flat = index.reshape(-1)
    count = torch.zeros(weight.shape[0], device=grad.device, dtype=torch.float64).index_add_(
        0, flat, known.reshape(-1).double())
    rows = grad.shape[-1]
    grad_weight = torch.zeros(weight.shape, device=grad.device, dtype=torch.float64).index_add_(0, flat, kept.reshape(-1, rows))
    size = torch.zeros(weight.shape, device=grad.device, dtype=torch.float64).index_add_(0, flat, kept.abs().reshape(-1, rows))
    outs = [out, grad_weight * scale]
    bounds = [bound, (count + 2)[:, None] * U32 * size * abs(scale)]
    if positions is not None:
        length = tokens.shape[-1]
        per = grad.reshape(-1, length, rows)
        grad_positions = torch.zeros(positions.shape, device=grad.device, dtype=torch.float64)
        grad_positions[:length] = per.sum(0)
        size = torch.zeros_like(grad_positions)
        size[:length] = per.abs().sum(0)
        outs.append(grad_positions)
        bounds.append((per.shape[0] + 1) * U32 * size)
    return outs, bounds


def loss(hidden, weight, targets, ignore_index, reduction, grad, recompute=False):
    """(loss, dH, dW) and bounds.

    A logit adds D products, exact in FP32 for 16-bit inputs: off by at most D roundings of
    sum |h w|.  FP32 inputs are two FP16 numbers each: every product is off by at most 4
    more units of 2^-24, and a value below 2^-40 of its tensor's largest is lost.  P is off by twice the logits'
    error (its own and the sum's), 16 roundings of the exponential, the reciprocal and the factors,
    and its storage: half a step of the operands' type (FP32: of 24 bits), or 2^-39 of
    the largest upstream gradient where FP16 runs out of exponents.

    Without `recompute` the exponentials of BF16 inputs have been rounded to FP16 before: relative to the largest of
    128, which is at most 2^15.5 then, off by 2^-11 of their own or, below the normal numbers, by 2^-25; so a
    probability is off by 2^-11 of its own or by 2^-25 / 2^15 times at most 2^1.5 (the references are off by half a power of two
    from either's largest).
    """
    dtype = hidden.dtype
    width, vocab = weight.shape[1], weight.shape[0]
    h, w = hidden.double().reshape(-1, width), weight.double()
    t = targets.reshape(-1)
    kept = t != ignore_index
    h = torch.where(kept[:, None], h, 0.0)  # what an ignored row holds is not looked at
    index = torch.where(kept, t, 0).long()
    logits = h @ w.T
    magnitude = h.abs() @ w.abs().T
    off = (width + 8) * U32 * magnitude.amax(-1, keepdim=True)
    if dtype == torch.float32:
        off = off + 2.0**-40 * (h.abs().amax() * w.abs().sum(-1).amax() + w.abs().amax() * h.abs().sum(-1, keepdim=True))
    lse = torch.logsumexp(logits, -1, keepdim=True)
    losses = torch.where(kept, (lse - logits.gather(1, index[:, None])).squeeze(1), 0.0)
    spread = (logits - logits.amax(-1, keepdim=True)).abs().amax(-1, keepdim=True)
    each = torch.where(kept, (2 * off + 16 * U32 * (1 + spread + lse.abs())).squeeze(1), 0.0)
    grad = grad.double().reshape(-1)
    if reduction == "none":
        out, bound, upstream = losses.view(targets.shape), each.view(targets.shape), grad
    elif reduction == "sum":
        out, upstream = losses.sum(), grad.expand(len(t))
        bound = each.sum() + 32 * U32 * losses.abs().sum() + len(t) / 1024 * U32 * losses.abs().sum()
    else:
        out, upstream = losses.sum() / kept.sum(), grad.expand(len(t)) / kept.sum()
        bound = (each.sum() + (34 + len(t) / 1024) * U32 * losses.abs().sum()) / kept.sum()
    upstream = torch.where(kept, upstream, 0.0)
    p = torch.softmax(logits, -1)
    soft = p * upstream.abs()[:, None]
    p = p.scatter_add(1, index[:, None], torch.full_like(p[:, :1], -1.0)) * upstream[:, None]
    off_p = soft * (2 * off + 16 * U32 * (1 + spread)) + HALF_STEP[dtype] * p.abs() + 4 * U32 * p.abs()
    # FP32 and BF16 end at 2^-126: an exponential below that is lost (times the upstream gradient), and so is a
    # row's factor times a probability below it (over a power of two of at most twice the largest
    # upstream gradient); three such losses stay below 2^-124 of that gradient
    off_p = off_p + 2.0**-124 * upstream.abs().amax() * kept[:, None]
    if dtype == torch.bfloat16 and not recompute:
        off_p = off_p + (1 + HALF_STEP[dtype]) * 2.0**-11 * soft
    if dtype != torch.bfloat16 or not recompute:
        off_p = off_p + 2.0**-38 * upstream.abs().amax() * kept[:, None]
    k = 16 * U32  # factors of the outputs, splits and pieces
    grad_hidden, grad_weight = p @ w, p.T @ h
    bound_h = off_p @ w.abs() + (vocab * U32 + k) * (p.abs() @ w.abs())
    bound_w = off_p.T @ h.abs() + (len(t) * U32 + k) * (p.abs().T @ h.abs())
    if dtype == torch.float32:
        bound_h = bound_h + 2.0**-40 * w.abs().amax() * p.abs().sum(-1, keepdim=True)
        bound_w = bound_w + 2.0**-40 * h.abs().amax() * p.abs().sum(0)[:, None]
    return ((out, grad_hidden.view(hidden.shape), grad_weight), (bound, bound_h.view(hidden.shape), bound_w))


__all__ = ["FLOOR", "HALF_STEP", "U32", "assert_within", "embedding", "layer_norm", "loss"]
