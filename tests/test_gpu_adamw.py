"""The AdamW step (attnres.optim) on the GPU against its FP64 definition
(tests/adamw_reference.py, where the bounds are derived): sizes around the edges of blocks and
workgroups, types, layouts, many tensors, values where a state could go wrong, graphs, and
the optimizer class around it."""

from __future__ import annotations

import copy
import io

import pytest
import torch

import adamw_reference as reference
from adamw_reference import assert_rounded, decoded
from attnres import layers, optim
from benchmarks.model import TrainingConfig, make_model, training_step
from layer_reference import FLOOR, HALF_STEP, assert_within

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
OPTIONS = dict(step=7, lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _quantised(values, least):
    """8-bit states of dense values, elements as they lie."""
    flat = values.as_strided((values.numel(),), (1,))
    blocks = -(-flat.numel() // 256)
    padded = torch.zeros(blocks * 256, device="cuda")
    padded[:flat.numel()] = flat
    scale = padded.view(blocks, 256).abs().amax(1) / 448
    numbers = padded.view(blocks, 256) / torch.where(scale > 0, scale, 1.0)[:, None]
    numbers = torch.where(numbers > 0, numbers.clamp_min(least), numbers) if least else numbers
    held = torch.empty_like(values, dtype=torch.float8_e4m3fn)
    held.as_strided((flat.numel(),), (1,)).copy_(numbers.view(-1)[:flat.numel()].to(torch.float8_e4m3fn))
    return held, scale


def _inputs(seed, shapes, dtype, grad_dtype, bits, masters):
    g = _generator(seed)

    def randn(shape):
        return torch.randn(shape, generator=g, device="cuda")

    state = {k: [] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales", "masters")}
    for shape in shapes:
        spread = 1e-3 * torch.exp(2 * randn(shape))
        weight, mean, root = 0.05 * randn(shape), 0.3 * spread * randn(shape), spread * (0.5 + torch.rand(shape, generator=g, device="cuda"))
        state["params"].append(weight.to(dtype))
        state["masters"].append(weight)
        state["grads"].append((spread * randn(shape)).to(grad_dtype))
        if bits == 8:
            for name, values, least in (("exp_avg", mean, 0.0), ("exp_avg_sq", root, 2.0**-9)):
                numbers, scale = _quantised(values, least)
                state[name + "s"].append(numbers)
                state[name + "_scales"].append(scale)
        else:
            state["exp_avgs"].append(mean)
            state["exp_avg_sqs"].append(root.square())
    if bits != 8:
        state["exp_avg_scales"] = state["exp_avg_sq_scales"] = None
    if not masters:
        state["masters"] = None
    return state


def _copy(state):
    return {k: None if v is None else [torch.empty_like(t).copy_(t) for t in v] for k, v in state.items()}


def _states(state, i):
    """(m, v) that the states of tensor i stand for."""
    m, v = state["exp_avgs"][i], state["exp_avg_sqs"][i]
    if state["exp_avg_scales"] is None:
        return m, v
    return decoded(m, state["exp_avg_scales"][i]), decoded(v, state["exp_avg_sq_scales"][i]).square()


def _check(state, grad_scale=None, **options):
    options = {**OPTIONS, **options}
    before = _copy(state)
    optim.adamw_step(**state, grad_scale=grad_scale, **options)
    for i, p in enumerate(state["params"]):
        source = p if state["masters"] is None else state["masters"][i]
        weight = before["params" if state["masters"] is None else "masters"][i]
        assert torch.equal(state["grads"][i], before["grads"][i])
        (w, m, v), (off_w, off_m, off_v) = reference.step(weight, before["grads"][i], *_states(before, i), grad_scale=grad_scale,
                                                          **{k: options[k] for k in OPTIONS})
        if state["masters"] is not None:
            assert torch.equal(p, source.to(p.dtype))
        assert_within(f"w[{i}]", source, w, off_w)
        if state["exp_avg_scales"] is None:
            assert_within(f"m[{i}]", state["exp_avgs"][i], m, off_m)
            assert_within(f"v[{i}]", state["exp_avg_sqs"][i], v, off_v)
        else:
            assert_rounded(f"m[{i}]", state["exp_avgs"][i], state["exp_avg_scales"][i], m, off_m)
            root = v.sqrt()
            off = torch.where(root > 0, off_v / root.clamp_min(1e-300), 0.0).minimum(off_v.sqrt()) + reference.K * root
            assert_rounded(f"v[{i}]", state["exp_avg_sqs"][i], state["exp_avg_sq_scales"][i], root, off, root=True)
    return state


SHAPES = [(1,), (3,), (255,), (256,), (257,), (64, 33), (1024,), (4095,), (4096,), (4097,), (0,), (7, 5, 300), (300, 1000)]
KINDS = [(FP32, FP32, False), (BF16, BF16, False), (BF16, BF16, True), (BF16, FP32, True), (FP16, FP16, True), (FP16, FP16, False),
         (FP16, FP32, False)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,grad_dtype,masters", KINDS)
def test_step(dtype, grad_dtype, masters, bits):
    _check(_inputs(1, SHAPES, dtype, grad_dtype, bits, masters))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 55, 56, 57, 113])
def test_more_tensors_than_a_launch_takes(count, bits):
    _check(_inputs(count, [(1 + 97 * k % 1500,) for k in range(count)], FP32, FP32, bits, False))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_large_tensor_among_small_ones(bits):
    _check(_inputs(3, [(5,), (3000, 1111), (70000,), (1,)], BF16, BF16, bits, True))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("options", [dict(step=1), dict(step=2**40), dict(betas=(0.0, 0.0)), dict(betas=(0.9, 0.999), step=100000),
                                     dict(weight_decay=0.0), dict(lr=0.0), dict(eps=1e-3)])
def test_factors(options, bits):
    _check(_inputs(4, [(1000,), (130,)], FP32, FP32, bits, False), **options)


@pytest.mark.parametrize("bits", [32, 8])
def test_factors_on_the_device(bits):
    state = _inputs(5, [(1000,), (130,)], FP32, FP32, bits, False)
    other = _copy(state)
    scale = torch.tensor(0.3, device="cuda")
    optim.adamw_step(**state, grad_scale=scale, **{**OPTIONS, "lr": float(torch.tensor(3e-3))})
    optim.adamw_step(**other, grad_scale=scale, **{**OPTIONS, "step": torch.tensor([7], device="cuda"),
                                                   "lr": torch.tensor(3e-3, device="cuda")})
    for k, tensors in state.items():
        for a, b in zip(tensors or [], other[k] or []):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), k


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_gradient_scale(dtype, bits):
    _check(_inputs(6, [(1000,), (64, 65)], dtype, dtype, bits, dtype != FP32), grad_scale=torch.tensor([0.125], device="cuda"))


@pytest.mark.parametrize("bits", [32, 8])
def test_the_first_step_from_zero_states(bits):
    state = _inputs(7, [(3000,), (70,)], FP32, FP32, bits, False)
    for name in ("exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales"):
        for t in state[name] or []:
            t.zero_()
    _check(state, step=1)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_of_zero(bits):
    """Elements that have never had a gradient keep their states of zero, and only decay."""
    state = _inputs(8, [(1500,)], FP32, FP32, bits, False)
    zero = torch.arange(1500, device="cuda") % 3 == 0
    zero[512:768] = True
    state["grads"][0][zero] = 0.0
    for name in ("exp_avgs", "exp_avg_sqs"):
        held = state[name][0]
        state[name][0] = held.float().masked_fill(zero, 0.0).to(held.dtype)
    if bits == 8:
        state["exp_avg_scales"][0][2] = state["exp_avg_sq_scales"][0][2] = 0.0
    before = state["params"][0].clone()
    _check(state)
    assert not bool(state["exp_avgs"][0].float()[zero].any()) and not bool(state["exp_avg_sqs"][0].float()[zero].any())
    decayed = before * torch.tensor(1 - OPTIONS["lr"] * OPTIONS["weight_decay"], device="cuda")
    assert torch.equal(state["params"][0][zero], decayed[zero])


def test_small_roots_beside_large_ones_do_not_vanish():
    """A block whose gradients span 2^40: the smallest roots are held by the least number, so no update explodes."""
    magnitude = torch.exp2(-40.0 * torch.arange(512, device="cuda") / 512)
    state = {"params": [torch.zeros(512, device="cuda")], "grads": [magnitude], "masters": None}
    for name in ("exp_avg", "exp_avg_sq"):
        state[name + "s"] = [torch.zeros(512, device="cuda").to(torch.float8_e4m3fn)]
        state[name + "_scales"] = [torch.zeros(2, device="cuda")]
    for step in range(1, 4):
        before = state["params"][0].clone()
        _check(state, step=step, weight_decay=0.0, lr=1.0)
        # with gradients of one size a step is lr; m and the root have the same share of their block's largest, so both are
        # rounded alike, by 2^-4 at most while normal numbers last, and below that the root more upwards than m
        assert float((state["params"][0] - before).abs().max()) <= (1 + 2.0**-4) / (1 - 2.0**-4)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_gradients_that_are_not_finite(bad):
    for bits in (32, 8):
        state = _inputs(9, [(2000,)], FP32, FP32, bits, False)
        clean = _copy(state)
        optim.adamw_step(**clean, **OPTIONS)
        state["grads"][0][700] = bad
        optim.adamw_step(**state, **OPTIONS)
        others = torch.arange(2000, device="cuda") != 700
        assert torch.equal(state["params"][0][others], clean["params"][0][others])
        assert not bool(state["params"][0][700].isfinite())
        if bits == 32:
            for name in ("exp_avgs", "exp_avg_sqs"):
                assert torch.equal(state[name][0][others], clean[name][0][others]) and not bool(state[name][0][700].isfinite())
        else:
            away = torch.arange(2000, device="cuda") // 256 != 700 // 256
            for name in ("exp_avg", "exp_avg_sq"):
                values, expected = (decoded(s[name + "s"][0], s[name + "_scales"][0]) for s in (state, clean))
                assert torch.equal(values[away], expected[away]) and bool(values[~away].isnan().all())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_layouts(dtype, bits):
    """Views at any element of a buffer, transposed weights, gradients in another order, with gaps or one for all."""
    state = _inputs(10, [(37, 65), (50, 20), (10, 30), (2000,), (40, 16)], dtype, dtype, bits, dtype != FP32)
    plain = _copy(state)
    optim.adamw_step(**plain, **OPTIONS)

    def shifted(t):
        buffer = torch.empty(t.numel() + 3, dtype=t.dtype, device="cuda")
        return buffer[3:].view(t.shape).copy_(t)

    def gaps(t):
        return torch.empty(t.shape[0], t.shape[1] + 5, dtype=t.dtype, device="cuda")[:, 2:2 + t.shape[1]].copy_(t)

    for k, tensors in state.items():
        if tensors is not None:
            tensors[0] = shifted(tensors[0])
            tensors[3] = shifted(tensors[3])
    state["grads"][1] = state["grads"][1].T.contiguous().T
    state["grads"][2] = gaps(state["grads"][2])
    row = state["grads"][4][:1].clone()
    state["grads"][4] = row.expand(40, 16)
    again = _inputs(10, [(37, 65), (50, 20), (10, 30), (2000,), (40, 16)], dtype, dtype, bits, dtype != FP32)
    again["grads"][4] = row.expand(40, 16).contiguous()
    optim.adamw_step(**again, **OPTIONS)
    optim.adamw_step(**state, **OPTIONS)
    for k, tensors in state.items():
        for i, (a, b) in enumerate(zip(tensors or [], again[k] or [])):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), (k, i)
    for i in range(4):
        assert torch.equal(state["params"][i], plain["params"][i])


@pytest.mark.parametrize("bits", [32, 8])
def test_transposed_parameters(bits):
    state = _inputs(11, [(90, 70)], FP32, FP32, bits, False)
    turned = {k: None if v is None else [t if t.dim() == 1 else t.T for t in v] for k, v in _copy(state).items()}
    turned["grads"] = [turned["grads"][0].contiguous()]  # in the order of the transposed shape: copied
    optim.adamw_step(**state, **OPTIONS)
    optim.adamw_step(**turned, **OPTIONS)
    assert torch.equal(state["params"][0], turned["params"][0].T) and torch.equal(state["exp_avgs"][0].float(), turned["exp_avgs"][0].T.float())


def test_nothing_to_do():
    optim.adamw_step([], [], [], [], step=1, lr=0.1)
    empty = [torch.empty(0, 3, device="cuda")]
    optim.adamw_step(empty, [empty[0].clone()], [empty[0].clone()], [empty[0].clone()], step=1, lr=0.1)


def test_repeated_calls_and_another_stream_give_the_same_bits():
    state = _inputs(12, [(3000,), (129,)], BF16, BF16, 8, True)
    copies = [_copy(state) for _ in range(2)]
    optim.adamw_step(**state, **OPTIONS)
    optim.adamw_step(**copies[0], **OPTIONS)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        optim.adamw_step(**copies[1], **OPTIONS)
    stream.synchronize()
    for other in copies:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for k in state for a, b in zip(state[k], other[k]))


def test_overlapping_tensors_are_refused():
    base = torch.zeros(100, device="cuda")
    apart = [[torch.zeros(60, device="cuda") for _ in range(2)] for _ in range(3)]
    for params in ([base[:60], base[40:]], [base[:60], base[:60]]):
        with pytest.raises(ValueError, match="overlap"):
            optim.adamw_step(params, apart[0], apart[1], apart[2], step=1, lr=0.1)
    with pytest.raises(ValueError, match="overlap"):
        optim.adamw_step(apart[0], apart[1], apart[2], [apart[2][1], apart[2][0]], step=1, lr=0.1)
    with pytest.raises(ValueError, match="overlap"):
        optim.adamw_step(apart[0], [apart[0][0], apart[1][0]], apart[1][1:] + apart[2][:1], [base[:60], torch.zeros(60, device="cuda")],
                         step=1, lr=0.1)
    one = torch.ones(60, device="cuda")  # gradients are only read, and may be one tensor
    optim.adamw_step(apart[0], [one, one], apart[1], apart[2], step=1, lr=0.1)
    assert torch.equal(apart[0][0], apart[0][1])


def test_a_backward_that_needs_the_old_weights_is_refused():
    weight = torch.randn(32, 32, device="cuda", requires_grad=True)
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    loss = (x @ weight).square().sum()
    zeros = [torch.zeros(32, 32, device="cuda") for _ in range(3)]
    optim.adamw_step([weight], zeros[:1], zeros[1:2], zeros[2:], step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_inference_tensors():
    with torch.inference_mode():
        tensors = [torch.ones(40, device="cuda") for _ in range(4)]
        optim.adamw_step(*([t] for t in tensors), step=1, lr=0.1)
        assert bool(tensors[0].isfinite().all())


# ------------------------------------------------------------- the optimizer

def _parameters(seed, dtype=FP32):
    g = _generator(seed)
    return [torch.nn.Parameter((0.1 * torch.randn(s, generator=g, device="cuda")).to(dtype)) for s in ((64, 128), (130,), (17, 9, 5))]


def _set_gradients(parameters, seed):
    g = _generator(seed)
    for p in parameters:
        p.grad = (torch.randn(p.shape, generator=g, device="cuda") * 0.1).to(p.dtype)


def test_optimizer_follows_the_definition_in_double():
    """Ten steps in FP32: each is off by the bounds of one, with the errors of the states before it, which a step
    multiplies by less than one; K units per step of the largest magnitudes."""
    parameters = _parameters(20)
    twins = [torch.nn.Parameter(p.detach().double()) for p in parameters]
    options = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
    optimizer, twin = optim.AdamW(parameters, **options), torch.optim.AdamW(twins, **options)
    for step in range(10):
        _set_gradients(parameters, 100 + step)
        for p, q in zip(parameters, twins):
            q.grad = p.grad.double()
        optimizer.step()
        twin.step()
    for p, q in zip(parameters, twins):
        scale = float(q.detach().abs().max()) + 10 * options["lr"]
        assert float((p.detach().double() - q.detach()).abs().max()) <= 10 * 4 * reference.K * scale
        for name in ("exp_avg", "exp_avg_sq"):
            a, b = optimizer.state[p][name].double(), twin.state[q][name]
            assert float((a - b).abs().max()) <= 10 * reference.K * float(b.abs().max())


@pytest.mark.parametrize("kind", ["fp32", "8-bit", "masters", "capturable"])
def test_state_dicts_continue_where_they_were(kind):
    dtype = BF16 if kind == "masters" else FP32
    options = dict(lr=1e-2, state_bits=8 if kind in ("8-bit", "masters") else 32, masters=kind == "masters", capturable=kind == "capturable")
    parameters = _parameters(21, dtype)
    optimizer = optim.AdamW(parameters, **options)
    for step in range(3):
        _set_gradients(parameters, 200 + step)
        optimizer.step()
    buffer = io.BytesIO()
    torch.save(optimizer.state_dict(), buffer)
    buffer.seek(0)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in parameters]
    other = optim.AdamW(twins, lr=0.5)
    other.load_state_dict(torch.load(buffer, weights_only=True))
    copied, loaded = copy.deepcopy(optimizer.state_dict())["state"], other.state_dict()["state"]
    assert copied.keys() == loaded.keys()
    for index, state in copied.items():
        assert state.keys() == loaded[index].keys()
        assert all(loaded[index][k].dtype == v.dtype for k, v in state.items() if isinstance(v, torch.Tensor))
    for step in range(2):
        for ps in (parameters, twins):
            _set_gradients(ps, 300 + step)
        optimizer.step()
        other.step()
    for p, q in zip(parameters, twins):
        assert torch.equal(p, q)
        for name, value in optimizer.state[p].items():
            mine = other.state[q][name]
            assert int(mine) == int(value) if name == "step" else torch.equal(mine.view(torch.uint8), value.view(torch.uint8))
    assert int(optimizer.state[parameters[0]]["step"]) == 5
    if kind in ("8-bit", "masters"):
        assert optimizer.state[parameters[0]]["exp_avg"].dtype == torch.float8_e4m3fn  # 8192 elements
        assert optimizer.state[parameters[1]]["exp_avg"].dtype == FP32


def test_state_of_torch_adamw_loads():
    parameters = _parameters(22)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in parameters]
    theirs = torch.optim.AdamW(twins, lr=1e-2)
    for step in range(2):
        _set_gradients(twins, 400 + step)
        theirs.step()
    for p, q in zip(parameters, twins):
        p.data.copy_(q)
    mine = optim.AdamW(parameters, lr=1.0, state_bits=8)
    mine.load_state_dict(theirs.state_dict())
    for ps, optimizer in ((parameters, mine), (twins, theirs)):
        _set_gradients(ps, 500)
        optimizer.step()
    for p, q in zip(parameters, twins):
        assert mine.state[p]["step"] == 3
        # both FP32, a step of at most lr
        assert float((p - q).detach().abs().max()) <= 4 * reference.K * (float(q.detach().abs().max()) + 1e-2)


@pytest.mark.parametrize("capturable", [False, True])
def test_parameters_without_a_gradient_wait(capturable):
    parameters = _parameters(23)
    optimizer = optim.AdamW(parameters, lr=1e-2, capturable=capturable)
    counts = []
    for step, missing in enumerate((2, None, 1, 1, None)):
        _set_gradients(parameters, 600 + step)
        before = [p.detach().clone() for p in parameters]
        if missing is not None:
            parameters[missing].grad = None
        optimizer.step()
        for k, (p, old) in enumerate(zip(parameters, before)):
            assert torch.equal(p, old) == (k == missing)
    counts = [int(optimizer.state[p]["step"]) for p in parameters]
    assert counts == [5, 3, 4]


def test_groups_types_and_a_closure():
    wide, narrow = _parameters(24), _parameters(25, BF16)
    optimizer = optim.AdamW([{"params": wide + narrow, "lr": 1e-2}, {"params": _parameters(26), "weight_decay": 0.0}], lr=1e-3,
                            masters=True)
    everything = [p for group in optimizer.param_groups for p in group["params"]]
    _set_gradients(everything, 700)
    before = [p.detach().clone() for p in everything]
    assert optimizer.step(lambda: 3.5) == 3.5
    assert all(not torch.equal(p, q) for p, q in zip(everything, before))
    assert "master" not in optimizer.state[wide[0]] and optimizer.state[narrow[0]]["master"].dtype == FP32
    scheduler = torch.optim.lr_scheduler.StepLR(optimizer, 1, 0.5)
    optimizer.step()
    scheduler.step()
    assert optimizer.param_groups[0]["lr"] == 5e-3


def test_sixteen_bit_weights_move_with_masters():
    """Steps far below half a step of BF16: without masters they are lost, with them they add up."""
    moved = {}
    for masters in (False, True):
        p = torch.nn.Parameter(torch.ones(5000, device="cuda", dtype=BF16))
        optimizer = optim.AdamW([p], lr=1e-4, weight_decay=0.0, masters=masters)
        for _ in range(100):
            p.grad = torch.ones_like(p)
            optimizer.step()
        moved[masters] = float(1 - p.detach().float().mean())
    # every step moves by lr (m / sqrt(v) = 1 up to eps): 0.01 in all, rounded to BF16 below 1 (steps of 2^-8)
    assert moved[False] == 0.0 and abs(moved[True] - 0.01) <= 2.0**-9


def test_a_captured_training_step():
    """Weights, their gradients through the feed-forward block, and the step, captured; the learning rate changes
    between replays.  Every replay against the same steps run eagerly."""
    g = _generator(27)

    def make():
        gen = _generator(28)
        return [torch.nn.Parameter((0.1 * torch.randn(s, generator=gen, device="cuda")).to(BF16)) for s in ((192, 64), (64, 96))]

    x, target = torch.zeros(48, 64, device="cuda", dtype=BF16), torch.zeros(48, 64, device="cuda")
    batches = [(torch.randn(48, 64, generator=g, device="cuda").to(BF16), torch.randn(48, 64, generator=g, device="cuda")) for _ in range(4)]
    rate = torch.tensor(1e-2, device="cuda")
    results = []
    for captured in (False, True):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            weights = make()
            optimizer = optim.AdamW(weights, lr=rate, state_bits=8, masters=True, capturable=True)

            def step(weights=weights, optimizer=optimizer):
                out = layers.gated_feed_forward(x, *weights)
                loss = (out.float() - target).square().mean()
                for p, grad in zip(weights, torch.autograd.grad(loss, weights)):
                    p.grad.copy_(grad)
                optimizer.step()
                return loss.detach()

            for p in weights:
                p.grad = torch.zeros_like(p)
            x.copy_(batches[0][0]), target.copy_(batches[0][1])
            step()
        stream.synchronize()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                loss = step()
            # the capture ran nothing
        losses = []
        for k, batch in enumerate(batches[1:]):
            with torch.cuda.stream(stream):
                x.copy_(batch[0]), target.copy_(batch[1])
                rate.fill_(1e-2 / (k + 1))
                if captured:
                    graph.replay()
                    losses.append(loss.clone())
                else:
                    losses.append(step())
            torch.cuda.synchronize()
        rate.fill_(1e-2)
        results.append([*losses, *weights, *(v for p in weights for v in optimizer.state[p].values())])
    assert len(results[0]) == len(results[1])
    for a, b in zip(*results):
        assert torch.equal(a.detach().reshape(-1).view(torch.uint8), b.detach().reshape(-1).view(torch.uint8))
    assert int(results[0][5]) == 4  # the first weight's count of steps


def test_capture_is_refused_without_state_or_device_counts():
    for capturable in (False, True):
        p = torch.nn.Parameter(torch.ones(64, device="cuda"))
        p.grad = torch.ones_like(p)
        optimizer = optim.AdamW([p], capturable=capturable)
        if not capturable:
            optimizer.step()
        torch.cuda.synchronize()
        graph, scratch = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
        with torch.cuda.graph(graph):
            scratch.add_(1)
            with pytest.raises(RuntimeError, match="captur"):
                optimizer.step()


@pytest.mark.parametrize("state_bits", [32, 8])
def test_training_steps_of_the_model(state_bits):
    """The model with this package's layers and its optimizer against torch's AdamW on the same gradients."""
    config = TrainingConfig(layers=2, width=64, heads=4, ffn=96, batch=2, sequence=32, vocab=97)
    torch.manual_seed(29)
    model = make_model(config, source_bank=True, fused_layers=True).cuda()
    before = [p.detach().clone() for p in model.parameters()]
    optimizer = optim.AdamW(model.parameters(), lr=1e-3, state_bits=state_bits)
    tokens = torch.randint(config.vocab, (config.batch, config.sequence), device="cuda")
    training_step(model, optimizer, tokens, torch.roll(tokens, -1, dims=1), accumulation=2)
    for p, old in zip(model.parameters(), before):
        twin = torch.nn.Parameter(old.clone())
        twin.grad = p.grad.clone()
        torch.optim.AdamW([twin], lr=1e-3).step()
        # the first step: the weights depend on no rounded state
        assert float((p.detach() - twin.detach()).abs().max()) <= 4 * reference.K * (float(old.abs().max()) + 1e-3)
