"""State dicts of attnres.optim.AdamW on the GPU: steps after a load against those of an optimizer that had the
state from the start."""

from __future__ import annotations

import pytest
import torch

from attnres import optim

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_masters_of_a_loaded_state_without_them(dtype, capturable):
    """Torch's state, loaded with masters=True: the same steps as with the state's values and masters given to `adamw_step`;
    captured, refused until a step has made them."""
    p = torch.nn.Parameter(_randn(1, 70, 90).to(dtype))
    theirs = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone())], lr=1e-3)
    theirs.param_groups[0]["params"][0].grad = _randn(2, 70, 90).to(dtype)
    theirs.step()
    mine = optim.AdamW([p], lr=1e-5, weight_decay=0.0, masters=True, capturable=capturable)
    mine.load_state_dict({**theirs.state_dict(), "param_groups": mine.state_dict()["param_groups"]})
    saved = theirs.state_dict()["state"][0]
    param, mean, square, master = p.detach().clone(), saved["exp_avg"].float(), saved["exp_avg_sq"].float(), p.detach().float()
    p.grad = torch.zeros_like(p)
    if capturable:
        torch.cuda.synchronize()
        graph, scratch = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
        with torch.cuda.graph(graph):
            scratch.add_(1)
            with pytest.raises(RuntimeError, match="captur"):
                mine.step()
    for step in range(2, 5):
        p.grad = _randn(step + 1, 70, 90).to(dtype)
        mine.step()
        optim.adamw_step([param], [p.grad], [mean], [square], step=step, lr=1e-5, weight_decay=0.0, masters=[master])
    state = mine.state[p]
    assert int(state["step"]) == 4
    assert torch.equal(p, param) and torch.equal(state["exp_avg"], mean) and torch.equal(state["exp_avg_sq"], square)
    assert torch.equal(state["master"], master) and not torch.equal(master, param.float())


@pytest.mark.parametrize("capturable", [False, True])
def test_steps_that_are_refused_are_not_counted(capturable):
    """Of two groups the second one's parameter and state overlap: the first is stepped and counted, the second neither."""
    first, second = (torch.nn.Parameter(torch.ones(40, device="cuda").to(dtype)) for dtype in (BF16, FP32))
    optimizer = optim.AdamW([{"params": [first]}, {"params": [second]}], capturable=capturable)
    for p in (first, second):
        p.grad = torch.ones_like(p)
    optimizer.step()
    held = optimizer.state[second]["exp_avg"]
    optimizer.state[second]["exp_avg"] = second.detach()
    before = second.detach().clone()
    with pytest.raises(ValueError, match="overlap"):
        optimizer.step()
    assert [int(optimizer.state[p]["step"]) for p in (first, second)] == [2, 1]
    optimizer.state[second]["exp_avg"] = held
    assert torch.equal(second, before)
    optimizer.step()
    assert [int(optimizer.state[p]["step"]) for p in (first, second)] == [3, 2]


def test_a_refused_step_of_a_shared_count():
    """Parameters of two types share a count on the device; it is taken back where none of them was stepped."""
    first, second = (torch.nn.Parameter(torch.ones(40, device="cuda").to(dtype)) for dtype in (BF16, FP32))
    optimizer = optim.AdamW([first, second], capturable=True)
    for p in (first, second):
        p.grad = torch.ones_like(p)
    optimizer.step()
    assert optimizer.state[first]["step"] is optimizer.state[second]["step"]
    with pytest.raises(TypeError, match="grad_scale"):
        optimizer.step(grad_scale=torch.ones(1, device="cuda", dtype=BF16))
    assert int(optimizer.state[first]["step"]) == 1
    optimizer.step()
    assert int(optimizer.state[first]["step"]) == 2
