"""The model with the layers of attnres.layers against the same model with torch's:
the loss and every parameter gradient, in FP32 and under BF16 autocast, with and
without the source bank; and its training step."""

from __future__ import annotations

import pytest
import torch

from benchmarks.model import TrainingConfig, make_model, training_step
from oracle.oracle import oracle

pytestmark = pytest.mark.gpu


def _config(mode, vocab=97):
    return TrainingConfig(layers=3, width=64, heads=4, ffn=128, batch=2, sequence=32, vocab=vocab, block_count=2, mode=mode)


def _relative_error(a, b):
    return float((a - b).abs().max() / b.abs().max().clamp_min(1e-12))


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("source_bank", [False, True])
@pytest.mark.parametrize("mode", ["full", "block"])
def test_fused_layers_match_the_model_with_torch_layers(mode, source_bank, autocast):
    """FP32 outside the reads: the layers differ in FP32 rounding only, which moves the reads' BF16
    sources by an ulp now and then: the tolerance of the compiled model's comparison.  Under
    autocast torch's model also rounds its logits to BF16 before the loss (2^-8 of logits of
    about 1, twice: the logits and, in the backward, the probabilities), hence twice that."""
    config = _config(mode)
    torch.manual_seed(71)
    plain = make_model(config, source_bank=source_bank).cuda()
    fused = make_model(config, source_bank=source_bank, fused_layers=True).cuda()
    fused.load_state_dict(plain.state_dict())
    tokens = torch.randint(config.vocab, (config.batch, config.sequence), device="cuda")
    targets = torch.roll(tokens, -1, dims=1).masked_fill(torch.arange(config.sequence, device="cuda") % 5 == 4, -100)
    limit = 4e-2 if autocast else 2e-2
    losses = []
    for model in (plain, fused):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            loss = model.loss(tokens, targets)
        loss.backward()
        losses.append(loss.detach())
    assert _relative_error(losses[1], losses[0]) < limit
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        assert q.grad.dtype == p.grad.dtype and _relative_error(q.grad, p.grad) < limit, name
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        assert _relative_error(fused(tokens).float(), plain(tokens).float()) < limit


def test_fused_training_steps_run_with_accumulation():
    config = _config("full")
    torch.manual_seed(73)
    model = make_model(config, source_bank=True, fused_layers=True).cuda()
    before = [p.detach().clone() for p in model.parameters()]
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    tokens = torch.randint(config.vocab, (config.batch, config.sequence), device="cuda")
    for _ in range(2):
        loss = training_step(model, optimizer, tokens, torch.roll(tokens, -1, dims=1), accumulation=2)
    assert bool(loss.isfinite())
    assert all(bool(p.isfinite().all()) and not torch.equal(p, q) for p, q in zip(model.parameters(), before))


def test_fused_layers_with_compiled_sublayers():
    config = _config("full")
    torch.manual_seed(79)
    plain = make_model(config, source_bank=True, fused_layers=True).cuda()
    compiled = make_model(config, source_bank=True, fused_layers=True, compile_layers=True).cuda()
    compiled.load_state_dict(plain.state_dict())
    tokens = torch.randint(config.vocab, (config.batch, config.sequence), device="cuda")
    losses = [model.loss(tokens, tokens) for model in (plain, compiled)]
    for loss in losses:
        loss.backward()
    assert _relative_error(losses[1].detach(), losses[0].detach()) < 2e-2
    for (name, p), q in zip(plain.named_parameters(), compiled.named_parameters()):
        assert _relative_error(q[1].grad, p.grad) < 2e-2, name


def test_fused_layers_need_the_hip_backend():
    with pytest.raises(ValueError, match="HIP"):
        make_model(_config("full"), backend=oracle, fused_layers=True)
