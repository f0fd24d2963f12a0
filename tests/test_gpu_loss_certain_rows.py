"""The loss's gradient where the target's probability is near one: its entry of P is 1 - p, which has to be
as accurate relative to itself as the others are, not relative to p."""

from __future__ import annotations

import pytest
import torch

from attnres import layers
from layer_reference import HALF_STEP, U32, assert_within

pytestmark = pytest.mark.gpu


def _certain_rows(rows, width, vocab, dtype):
    """Rows along their target's row of the weight, so that 1 - p of the target goes from about 1e-2 to 1e-5.
    Entries are small multiples of 2^-4 and 2^-6: every sum of products is exact in FP32, so the logits are."""
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    weight = ((torch.randn(vocab, width, generator=g, device="cuda") * 4).round() / 16).clamp(-1, 1)
    targets = torch.randint(vocab, (rows,), generator=g, device="cuda")
    own = weight[targets]
    height = torch.linspace(11.5, 19.0, rows, device="cuda")[:, None]
    hidden = (own * (height / own.square().sum(-1, keepdim=True)) * 64).round() / 64
    assert torch.equal(hidden.to(dtype).float(), hidden) and torch.equal(weight.to(dtype).float(), weight)
    assert float((hidden.abs() @ weight.abs().T).max()) < 2**13  # in units of 2^-10: 23 bits
    return hidden.to(dtype), weight.to(dtype), targets


@pytest.mark.parametrize("recompute", [False, True])
@pytest.mark.parametrize("rows,width,vocab", [(300, 256, 700), (70, 250, 1500), (40, 256, 129)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gradients_of_certain_rows(rows, width, vocab, dtype, recompute):
    """P off the target: half a step of the type, 2^-11 for kept exponentials of BF16 inputs, the exponentials' FP32
    roundings (16 times 1 + the exponent).  On the target: p - 1 of p = a / (a + b), where a's own error
    moves p by that times 1 - p; a sum of at most 64 roundings in a row, the reciprocal and the factors 8 more, each
    2^-24 of p; then half a step of 1 - p.  FP16's probabilities end at 2^-39 of the upstream gradient."""
    hidden, weight, targets = _certain_rows(rows, width, vocab, dtype)
    leaves = (hidden.requires_grad_(True), weight.requires_grad_(True))
    out = layers.linear_cross_entropy(*leaves, targets, reduction="sum", recompute=recompute)
    grads = torch.autograd.grad(out, leaves)
    h, w, at = hidden.detach().double(), weight.detach().double(), targets[:, None]
    logits = h @ w.T
    own = logits.gather(1, at)
    others = logits.scatter(1, at, -torch.inf).logsumexp(-1, keepdim=True)
    rest = torch.sigmoid(others - own)  # 1 - p of the target
    assert float(rest.max()) > 1e-3 and float(rest.min()) < 1e-4
    p = torch.softmax(logits, -1).scatter(1, at, -rest)
    exponent = (logits - logits.amax(-1, keepdim=True)).abs().amax(-1, keepdim=True)
    step = HALF_STEP[dtype] + 4 * U32 + 16 * U32 * (1 + exponent)
    kept = 2.0**-11 if dtype == torch.bfloat16 and not recompute else 0.0
    off = p.abs() * (step + kept * (1 + HALF_STEP[dtype]))
    off = off.scatter(1, at, rest * step + 72 * U32) + 2.0**-38
    bound_h = off @ w.abs() + (vocab * U32 + 16 * U32) * (p.abs() @ w.abs())
    bound_w = off.T @ h.abs() + (rows * U32 + 16 * U32) * (p.abs().T @ h.abs())
    if dtype == torch.float32:  # operands as pairs of FP16 numbers
        bound_h = bound_h + 2.0**-40 * w.abs().amax() * p.abs().sum(-1, keepdim=True)
        bound_w = bound_w + 2.0**-40 * h.abs().amax() * p.abs().sum(0)[:, None]
    assert_within("dH", grads[0], p @ w, bound_h)
    assert_within("dW", grads[1], p.T @ h, bound_w)


def test_certain_rows_of_bf16_agree_with_recomputed_ones():
    """Kept and recomputed exponentials give the target's entry from the same logit and the same sum: what is left
    between them is the other entries' 2^-11, and two roundings to BF16."""
    hidden, weight, targets = _certain_rows(300, 256, 700, torch.bfloat16)
    hidden.requires_grad_(True)
    grads = [torch.autograd.grad(layers.linear_cross_entropy(hidden, weight, targets, reduction="sum", recompute=r), hidden)[0].double()
             for r in (False, True)]
    difference = (grads[0] - grads[1]).norm(dim=-1) / grads[1].norm(dim=-1)
    # a row is (1 - p) (a mean of the others' rows - the target's): 2^-8 + 2^-11 of each part, the target's row being
    # the larger part, so 4 times that covers both
    assert float(difference.max()) <= 4 * (2.0**-8 + 2.0**-11)
