"""State dicts of attnres.optim.AdamW on the CPU: what is loaded, what is kept and what is refused.
Nothing launches."""

from __future__ import annotations

import pytest
import torch

from attnres import optim

BF16, FP32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _parameter(dtype=FP32, shape=(96, 64)):
    return torch.nn.Parameter(torch.linspace(-1.0, 1.0, 96 * 64).reshape(shape).to(dtype))


def _torch_dict(dtype=FP32, kind=torch.optim.AdamW, **options):
    """Of torch's optimizer after a step."""
    p = _parameter(dtype)
    optimizer = kind([p], **options)
    p.grad = torch.full_like(p, 0.5)
    optimizer.step()
    return optimizer.state_dict()


def test_hooks_of_a_load_see_and_make_what_is_loaded():
    p = _parameter()
    optimizer = optim.AdamW([p])
    seen = []

    def before(_optimizer, state_dict):
        state = {index: {**state, "exp_avg": state["exp_avg"] + 7.0} for index, state in state_dict["state"].items()}
        return {**state_dict, "state": state, "param_groups": [{**group, "lr": 0.25} for group in state_dict["param_groups"]]}

    def after(optimizer):
        seen.append((optimizer.state[p]["exp_avg"].dtype, optimizer.state[p]["step"]))
        optimizer.state[p]["exp_avg_sq"].fill_(3.0)

    optimizer.register_load_state_dict_pre_hook(before)
    optimizer.register_load_state_dict_post_hook(after)
    saved = _torch_dict()
    for _ in range(2):  # a load leaves no hooks of its own
        optimizer.load_state_dict(saved)
        assert torch.equal(optimizer.state[p]["exp_avg"], saved["state"][0]["exp_avg"] + 7.0)
        assert bool((optimizer.state[p]["exp_avg_sq"] == 3.0).all()) and optimizer.param_groups[0]["lr"] == 0.25
    assert seen == [(FP32, 1)] * 2
    with pytest.raises(ValueError):  # another number of groups
        optimizer.load_state_dict({**saved, "param_groups": saved["param_groups"] * 2})
    optimizer.load_state_dict(saved)
    assert len(seen) == 3


@pytest.mark.parametrize("options,match", [(dict(maximize=True), "maximize"), (dict(amsgrad=True), "amsgrad"),
                                           (dict(differentiable=True), "differentiable"),
                                           (dict(decoupled_weight_decay=False, weight_decay=0.1), "decoupled")])
def test_options_that_the_step_does_not_have_are_refused(options, match):
    """From a state dict (which then leaves the optimizer as it was) and from a group."""
    p = _parameter()
    optimizer = optim.AdamW([p], lr=0.5)
    saved = _torch_dict()
    for make in (lambda: optimizer.load_state_dict({**saved, "param_groups": [{**saved["param_groups"][0], **options}]}),
                 lambda: optimizer.add_param_group({"params": [_parameter()], **options}),
                 lambda: optim.AdamW([{"params": [p], **options}])):
        with pytest.raises(ValueError, match=match):
            make()
    assert not optimizer.state and optimizer.param_groups[0]["lr"] == 0.5 and len(optimizer.param_groups) == 1
    with pytest.raises(ValueError, match="decoupled"):
        optimizer.load_state_dict(_torch_dict(kind=torch.optim.Adam, weight_decay=0.1))
    optimizer.load_state_dict(_torch_dict())
    optimizer.load_state_dict(_torch_dict(kind=torch.optim.Adam))  # no decay, so the same step
    assert optimizer.state[p]["step"] == 1


@pytest.mark.parametrize("options,error", [(dict(betas=(0.9, 1.5)), ValueError), (dict(state_bits=4), ValueError), (dict(masters=1), TypeError),
                                           (dict(lr=-1.0), ValueError)])
def test_options_of_loaded_groups_are_checked(options, error):
    optimizer = optim.AdamW([_parameter()], lr=0.5)
    saved = _torch_dict()
    with pytest.raises(error, match=next(iter(options))):
        optimizer.load_state_dict({**saved, "param_groups": [{**saved["param_groups"][0], **options}]})
    assert not optimizer.state and optimizer.param_groups[0]["lr"] == 0.5


def test_options_that_a_state_dict_does_not_name_stay_as_they_are():
    first, second = _parameter(), _parameter()
    optimizer = optim.AdamW([{"params": [first], "state_bits": 8, "masters": True}, {"params": [second]}], lr=0.5)
    theirs = torch.optim.AdamW([{"params": [_parameter()], "lr": 0.25}, {"params": [_parameter()]}], lr=0.125)
    optimizer.load_state_dict(theirs.state_dict())
    assert [(g["lr"], g["state_bits"], g["masters"]) for g in optimizer.param_groups] == [(0.25, 8, True), (0.125, 32, False)]
    mine = optim.AdamW([{"params": [first]}, {"params": [second], "state_bits": 8}], lr=0.75)
    optimizer.load_state_dict(mine.state_dict())  # what it names is loaded
    assert [(g["lr"], g["state_bits"], g["masters"]) for g in optimizer.param_groups] == [(0.75, 32, False), (0.75, 8, False)]


@pytest.mark.parametrize("dtype", [BF16, torch.float16, FP32])
def test_masters_that_a_state_dict_lacks_are_made_from_the_parameters_at_the_next_step(dtype):
    p = _parameter(dtype)
    optimizer = optim.AdamW([p], masters=True)
    optimizer.load_state_dict(_torch_dict(dtype))
    with torch.no_grad():
        p.copy_(torch.linspace(3.0, 4.0, p.numel()).reshape(p.shape))  # weights that are loaded after the optimizer
    p.grad = torch.zeros_like(p)
    with pytest.raises(RuntimeError, match="CUDA"):
        optimizer.step()
    state = optimizer.state[p]
    assert ("master" in state) == (dtype != FP32) and state["exp_avg"].dtype == FP32
    if dtype != FP32:
        assert state["master"].dtype == FP32 and torch.equal(state["master"], p.detach().float())


def _eighth_dict(p):
    """Of this optimizer with 8-bit states, made by hand: numbers as the parameter's elements lie, a scale per 256."""
    optimizer = optim.AdamW([p], state_bits=8)
    state = {"step": 3}
    for name in ("exp_avg", "exp_avg_sq"):
        state[name] = torch.empty_like(p, dtype=FP32).copy_(torch.arange(p.numel()).reshape(p.shape) % 400).to(FP8)
        state[name + "_scale"] = torch.arange(1.0, -(-p.numel() // 256) + 1)
    return {"state": {0: state}, "param_groups": optimizer.state_dict()["param_groups"]}


def test_8_bit_states_of_another_order_of_elements_are_refused():
    """Their scales are of 256 elements as they lie: in another order numbers would meet other blocks' scales."""
    rows, columns = _parameter(), torch.nn.Parameter(_parameter().detach().T.contiguous().T)
    assert rows.shape == columns.shape and rows.stride() != columns.stride()
    for saved, loaded in ((rows, columns), (columns, rows)):
        optimizer = optim.AdamW([loaded], lr=0.5)
        with pytest.raises(ValueError, match="order"):
            optimizer.load_state_dict(_eighth_dict(saved))
        assert not optimizer.state and optimizer.param_groups[0]["lr"] == 0.5
    for p in (rows, columns, torch.nn.Parameter(torch.zeros(1, 5000).as_strided((1, 5000), (7, 1)))):
        saved = _eighth_dict(p)
        optimizer = optim.AdamW([p])
        optimizer.load_state_dict(saved)
        for name, value in saved["state"][0].items():
            mine = optimizer.state[p][name]
            assert mine == value if name == "step" else torch.equal(mine.float(), value.float()) and mine.dtype == value.dtype
    wide = optim.AdamW([columns])
    wide.load_state_dict(_torch_dict())  # 32-bit states have no blocks
    assert wide.state[columns]["exp_avg"].stride() == columns.stride()


@pytest.mark.parametrize("name,shape", [("exp_avg", (64,)), ("exp_avg_sq", (1, 64)), ("exp_avg", ()), ("master", (96, 1))])
def test_states_of_another_shape_are_refused(name, shape):
    """Also shapes that a copy would broadcast."""
    p = _parameter(BF16)
    saved = _torch_dict(BF16)
    saved["state"][0][name] = torch.ones(shape)
    optimizer = optim.AdamW([p], lr=0.5, masters=True)
    with pytest.raises(ValueError, match="shape"):
        optimizer.load_state_dict(saved)
    assert not optimizer.state and optimizer.param_groups[0]["lr"] == 0.5


def test_steps_that_are_refused_are_not_counted():
    """On the CPU every step is; so is one that meets a sparse gradient after others."""
    first, second = _parameter(), _parameter()
    optimizer = optim.AdamW([first, second])
    theirs = torch.optim.AdamW([_parameter(), _parameter()])
    for p in theirs.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    theirs.step()
    optimizer.load_state_dict(theirs.state_dict())
    first.grad = second.grad = torch.ones_like(first)
    with pytest.raises(RuntimeError, match="CUDA"):
        optimizer.step()
    second.grad = torch.ones_like(second).to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        optimizer.step()
    assert [optimizer.state[p]["step"] for p in (first, second)] == [1, 1]
