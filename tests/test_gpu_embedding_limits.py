"""The largest embedding gradient that the checks admit: its launches stay below 2^32 threads."""

from __future__ import annotations

import pytest
import torch

from attnres import layers

pytestmark = pytest.mark.gpu


def test_gradients_of_as_many_tokens_and_positions_as_there_may_be():
    """2^29 tokens and 2^26 rows of positions in one backward: 2^23 workgroups for the runs, and as many again if the positions
    took one for 8 rows.  Gradients are 1, 2 or 3, so that every sum here is exact."""
    batch, length, vocab = 8, 2**26, 2**16
    places = torch.arange(length, device="cuda", dtype=torch.int32)
    tokens = (places % vocab).expand(batch, length).contiguous()
    weight = torch.zeros(vocab, 1, device="cuda", requires_grad=True)
    positions = torch.zeros(length, 1, device="cuda", requires_grad=True)
    out = layers.embedding(tokens, weight, positions, dtype=torch.bfloat16)
    grad = (1 + places % 3).to(torch.bfloat16)[None, :, None].expand(batch, length, 1).contiguous()
    grad_weight, grad_positions = torch.autograd.grad(out, (weight, positions), grad)
    assert torch.equal(grad_positions[:, 0], batch * (1.0 + places % 3))
    # a word's places are 2^16 apart, so their gradients go round 1, 2, 3
    expected = batch * (1.0 + places % 3).view(length // vocab, vocab).sum(0)
    assert torch.equal(grad_weight[:, 0], expected)
