"""The model with its MLP sublayers as `attnres.layers.gated_feed_forward` and its weights
updated by `attnres.optim.AdamW`: against the same model with torch's, in FP32 and under BF16
autocast, compiled sublayers, and a whole captured training step."""

from __future__ import annotations

import copy

import pytest
import torch

from attnres.optim import AdamW
from benchmarks.model import TrainingConfig, make_model, training_step
from oracle.oracle import oracle

pytestmark = pytest.mark.gpu


def _config(mode="full"):
    return TrainingConfig(layers=3, width=64, heads=4, ffn=128, batch=2, sequence=32, vocab=97, block_count=2, mode=mode)


def _relative_error(a, b):
    return float((a - b).abs().max() / b.abs().max().clamp_min(1e-12))


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("fused_layers", [False, True])
@pytest.mark.parametrize("mode", ["full", "block"])
def test_fused_feed_forward_matches_the_model_with_torch_projections(mode, fused_layers, autocast):
    """FP32 outside the reads: FP32 rounding only, which moves the reads' BF16 sources by an ulp now and then: the tolerance
    of the compiled model's comparison.  Under autocast torch also rounds both projections and what the activation gives to
    BF16, 2^-8 each, in the forward and the backward: hence twice that."""
    config = _config(mode)
    torch.manual_seed(91)
    plain = make_model(config, source_bank=True, fused_layers=fused_layers).cuda()
    fused = make_model(config, source_bank=True, fused_layers=fused_layers, fused_feed_forward=True).cuda()
    fused.load_state_dict(plain.state_dict())
    tokens = torch.randint(config.vocab, (config.batch, config.sequence), device="cuda")
    targets = torch.roll(tokens, -1, dims=1)
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
        one = tokens[:1, :1]  # a single token
        assert _relative_error(fused(one).float(), plain(one).float()) < limit


def test_fused_feed_forward_with_compiled_sublayers():
    config = _config()
    torch.manual_seed(93)
    plain = make_model(config, source_bank=True, fused_layers=True, fused_feed_forward=True).cuda()
    compiled = make_model(config, source_bank=True, fused_layers=True, fused_feed_forward=True, compile_layers=True).cuda()
    compiled.load_state_dict(plain.state_dict())
    tokens = torch.randint(config.vocab, (config.batch, config.sequence), device="cuda")
    losses = []
    for model in (plain, compiled):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            losses.append(model.loss(tokens, tokens))
        losses[-1].backward()
    assert _relative_error(losses[1].detach(), losses[0].detach()) < 2e-2
    for (name, p), q in zip(plain.named_parameters(), compiled.named_parameters()):
        assert _relative_error(q[1].grad, p.grad) < 2e-2, name


def test_fused_feed_forward_needs_the_hip_backend():
    with pytest.raises(ValueError, match="HIP"):
        make_model(_config(), backend=oracle, fused_feed_forward=True)


@pytest.mark.parametrize("dtype,masters,state_bits", [(torch.float32, False, 32), (torch.float32, False, 8), (torch.bfloat16, True, 8)])
def test_training_steps_with_accumulation(dtype, masters, state_bits):
    config = _config()
    torch.manual_seed(95)
    model = make_model(config, source_bank=True, fused_layers=True, fused_feed_forward=True).cuda().to(dtype)
    before = [p.detach().clone() for p in model.parameters()]
    optimizer = AdamW(model.parameters(), lr=1e-2, state_bits=state_bits, masters=masters)
    tokens = torch.randint(config.vocab, (config.batch, config.sequence), device="cuda")
    for _ in range(3):
        loss = training_step(model, optimizer, tokens, torch.roll(tokens, -1, dims=1), accumulation=2)
    assert bool(loss.isfinite())
    assert all(bool(p.isfinite().all()) and not torch.equal(p, q) for p, q in zip(model.parameters(), before))
    assert all(optimizer.state[p]["step"] == 3 and ("master" in optimizer.state[p]) == masters for p in model.parameters())


@pytest.mark.parametrize("state_bits", [32, 8])
def test_captured_training_step_matches_compiled_steps(state_bits):
    """A whole step in one HIP graph, forward, backward and update: replays on changed batches against the same steps
    run eagerly from the same start (the tolerances of the same test with torch's optimizer; with 8-bit states a number on
    the border between two may fall to either side of it, which moves a weight by a part of a step of 1e-3)."""
    from benchmarks.training_graph import _loss, _step, capture_training_step

    config = _config()
    torch.manual_seed(97)
    model = make_model(config, fused_feed_forward=True).cuda()
    twin = copy.deepcopy(model)
    optimizer = AdamW(model.parameters(), lr=1e-3, state_bits=state_bits, capturable=True)
    twin_optimizer = AdamW(twin.parameters(), lr=1e-3, state_bits=state_bits, capturable=True)
    batches = [(torch.randint(config.vocab, (2 * config.batch, config.sequence), device="cuda"),
                torch.randint(config.vocab, (2 * config.batch, config.sequence), device="cuda")) for _ in range(3)]
    torch._dynamo.reset()
    captured = capture_training_step(model, optimizer, *batches[0], accumulation=2)
    assert all(int(optimizer.state[p]["step"]) == 0 for p in model.parameters())
    twin_model = torch.compile(twin, fullgraph=True, dynamic=False)
    twin_loss = torch.compile(_loss, fullgraph=True, dynamic=False)
    for index, (tokens, targets) in enumerate(batches):
        captured.copy_inputs(tokens, targets)
        loss = captured.replay().clone()
        expected = _step(twin_model, twin_loss, twin_optimizer, tokens, targets, 2)
        torch.cuda.synchronize()
        torch.testing.assert_close(loss, expected.detach(), rtol=1e-4, atol=1e-5, msg=f"step {index}")
    for (name, p), q in zip(model.named_parameters(), twin.parameters()):
        torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-6 if state_bits == 32 else 1e-4, msg=name)
    assert all(int(optimizer.state[p]["step"]) == 3 for p in model.parameters())


def test_a_captured_step_of_sixteen_bit_weights_starts_from_them():
    """Masters made while the capture warms up are set back to the weights, not to zeros."""
    from benchmarks.training_graph import capture_training_step

    config = _config()
    torch.manual_seed(99)
    model = make_model(config, fused_feed_forward=True).cuda().to(torch.bfloat16)
    before = [p.detach().clone() for p in model.parameters()]
    optimizer = AdamW(model.parameters(), lr=1e-3, masters=True, capturable=True)
    tokens = torch.randint(config.vocab, (config.batch, config.sequence), device="cuda")
    torch._dynamo.reset()
    captured = capture_training_step(model, optimizer, tokens, tokens)
    assert all(torch.equal(optimizer.state[p]["master"], q.float()) and torch.equal(p, q) for p, q in zip(model.parameters(), before))
    for _ in range(2):
        loss = captured.replay()
    torch.cuda.synchronize()
    assert bool(loss.isfinite())
    # two steps of at most 1e-3 each, and the decay of 1e-5
    for p, q in zip(model.parameters(), before):
        assert float((optimizer.state[p]["master"] - q.float()).abs().max()) <= 2.1e-3
