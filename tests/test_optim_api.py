"""The optimizer's public functions and C ABI on the CPU: refusals, and the binding against the header.
Nothing launches."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from attnres import _native, optim
from test_native_abi import _C_TYPES

HEADER = Path(__file__).resolve().parents[1] / "include" / "attnres_optim_hip.h"
BF16, FP16, FP32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _step(params=None, grads=None, exp_avgs=None, exp_avg_sqs=None, shape=(6, 50), dtype=FP32, bits=32, **kw):
    zeros = lambda kind, s=shape: [torch.zeros(s).to(kind)]  # noqa: E731
    state = FP8 if bits == 8 else FP32
    if bits == 8:
        for name in ("exp_avg_scales", "exp_avg_sq_scales"):
            kw.setdefault(name, zeros(FP32, (2,)))
    return optim.adamw_step(params if params is not None else zeros(dtype), grads if grads is not None else zeros(dtype),
                            exp_avgs if exp_avgs is not None else zeros(state), exp_avg_sqs if exp_avg_sqs is not None else zeros(state),
                            **{"step": 1, "lr": 0.1, **kw})


@pytest.mark.parametrize("kw", [{}, dict(bits=8), dict(dtype=BF16), dict(dtype=FP16, masters=[torch.zeros(6, 50)]),
                                dict(step=torch.tensor(1), lr=torch.tensor(0.1), grad_scale=torch.tensor(1.0)),
                                dict(dtype=BF16, grads=[torch.zeros(6, 50)])])
def test_cpu_tensors_are_refused_after_everything_else(kw):
    with pytest.raises(RuntimeError, match="CUDA"):
        _step(**kw)


def _apart(t):
    return torch.zeros(t, 2)[:, 0]


@pytest.mark.parametrize("kw,error,match", [
    (dict(params=[1.0]), TypeError, None),
    (dict(params=[]), ValueError, "as many grads"),
    (dict(grads=[]), ValueError, "as many grads"),
    (dict(exp_avgs=[]), ValueError, "as many exp_avgs"),
    (dict(exp_avg_sqs=[torch.zeros(6, 50)] * 2), ValueError, "as many exp_avg_sqs"),
    (dict(bits=8, exp_avg_scales=[]), ValueError, "as many exp_avg_scales"),
    (dict(masters=[], dtype=BF16), ValueError, "as many masters"),
    (dict(exp_avg_scales=[torch.zeros(2)]), ValueError, "go together"),
    (dict(dtype=torch.float64), TypeError, "params must be BF16"),
    (dict(grads=[torch.zeros(6, 50, dtype=torch.int64)]), TypeError, "grads must be BF16"),
    (dict(grads=[torch.zeros(6, 50, dtype=BF16)]), TypeError, "dtype of params or FP32"),
    (dict(dtype=BF16, grads=[torch.zeros(6, 50, dtype=FP16)]), TypeError, "dtype of params or FP32"),
    (dict(masters=[torch.zeros(6, 50)]), TypeError, "masters"),
    (dict(grads=[torch.zeros(50, 6)]), ValueError, "shape of its parameter"),
    (dict(grads=[torch.zeros(6, 50).to_sparse()]), TypeError, "dense"),
    (dict(exp_avgs=[torch.zeros(50, 6)]), ValueError, "shape and strides"),
    (dict(exp_avgs=[torch.zeros(50, 6).T]), ValueError, "shape and strides"),
    (dict(exp_avg_sqs=[torch.zeros(6, 50, dtype=BF16)]), TypeError, "exp_avg_sqs"),
    (dict(bits=8, exp_avgs=[torch.zeros(6, 50)]), TypeError, "exp_avgs"),
    (dict(dtype=BF16, masters=[torch.zeros(6, 50, dtype=BF16)]), TypeError, "masters"),
    (dict(dtype=BF16, masters=[torch.zeros(50, 6).T]), ValueError, "masters"),
    (dict(bits=8, exp_avg_scales=[torch.zeros(1)]), ValueError, "256"),
    (dict(bits=8, exp_avg_sq_scales=[_apart(2)]), ValueError, "256"),
    (dict(bits=8, exp_avg_scales=[torch.zeros(2, dtype=torch.float64)]), TypeError, "scales"),
    (dict(params=[torch.zeros(6, 100)[:, ::2]]), ValueError, "dense"),
    (dict(params=[torch.zeros(6, 1).expand(6, 50)]), ValueError, "dense"),
    (dict(grads=[torch.zeros(6, 50, device="meta")]), TypeError, "device"),
    (dict(step=0), ValueError, "step"),
    (dict(step=1.0), TypeError, "step"),
    (dict(step=True), TypeError, "step"),
    (dict(step=torch.tensor(1.0)), TypeError, "step"),
    (dict(step=torch.tensor([1, 2])), ValueError, "step"),
    (dict(lr=-0.1), ValueError, "lr"),
    (dict(lr=float("nan")), ValueError, "lr"),
    (dict(lr="0.1"), TypeError, "lr"),
    (dict(lr=torch.tensor(0.1, dtype=torch.float64)), TypeError, "lr"),
    (dict(betas=(0.9,)), TypeError, "betas"),
    (dict(betas=(0.9, 1.0)), ValueError, "betas"),
    (dict(betas=(-0.1, 0.9)), ValueError, "betas"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(weight_decay=float("inf")), ValueError, "weight_decay"),
    (dict(grad_scale=0.5), TypeError, "grad_scale"),
    (dict(grad_scale=torch.zeros(2)), ValueError, "grad_scale"),
    (dict(grad_scale=torch.zeros(1, dtype=BF16)), TypeError, "grad_scale"),
])
def test_refusals(kw, error, match):
    with pytest.raises(error, match=match):
        _step(**kw)


def test_tensors_of_several_types_are_refused():
    lists = [[torch.zeros(4), torch.zeros(4, dtype=BF16)], [torch.zeros(4), torch.zeros(4, dtype=BF16)], [torch.zeros(4)] * 2,
             [torch.zeros(4)] * 2]
    with pytest.raises(TypeError, match="one dtype"):
        optim.adamw_step(*lists, step=1, lr=0.1)
    with pytest.raises(TypeError, match="one dtype"):
        optim.adamw_step([torch.zeros(4, dtype=BF16)] * 2, *lists[1:], step=1, lr=0.1)


@pytest.mark.parametrize("kw,error", [
    (dict(lr=-1.0), ValueError), (dict(betas=(0.9, 1.0)), ValueError), (dict(eps=-1.0), ValueError), (dict(weight_decay=-1.0), ValueError),
    (dict(state_bits=16), ValueError), (dict(masters=1), TypeError), (dict(capturable=None), TypeError)])
def test_optimizer_refusals(kw, error):
    with pytest.raises(error):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)


def test_options_of_a_group_are_checked():
    first, second = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([{"params": [first], "state_bits": 4}])
    optimizer = optim.AdamW([first])
    with pytest.raises(ValueError, match="betas"):
        optimizer.add_param_group({"params": [second], "betas": (0.9, 1.5)})
    optimizer.add_param_group({"params": [second], "lr": 0.5, "masters": True})
    assert optimizer.param_groups[1]["lr"] == 0.5 and optimizer.param_groups[1]["fused"]


def test_optimizer_needs_gpu_parameters_and_dense_gradients():
    p = torch.nn.Parameter(torch.zeros(3, 4))
    optimizer = optim.AdamW([p])
    optimizer.step()  # no gradient, nothing to do
    p.grad = torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        optimizer.step()
    p.grad = torch.zeros(3, 4).to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        optimizer.step()


def test_binding_matches_the_header():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = dict(re.findall(r"\bint (attnres_hip_\w+)\(([^;]*)\);", text))
    assert set(declared) == set(_native.OPTIM_SIGNATURES)
    types = {**_C_TYPES, "double": ctypes.c_double, "const struct attnres_adamw_tensor*": ctypes.c_void_p}
    for name, arguments in declared.items():
        words = [re.sub(r"\s*\b\w+$", "", re.sub(r"\s+", " ", a.strip())).replace(" *", "*") for a in arguments.split(",")]
        assert _native.OPTIM_SIGNATURES[name][1] == [types[w] for w in words], name
    body = re.search(r"struct attnres_adamw_tensor \{(.*?)\};", text, re.S).group(1)
    fields = re.findall(r"(\w+);", body)
    assert fields == [name for name, _ in _native.AdamwTensor._fields_] and ctypes.sizeof(_native.AdamwTensor) == 64


def _abi(tensor=None, count=1, param_dtype=2, grad_dtype=2, bits=32, lr=0.1, beta1=0.9, beta2=0.9, eps=1e-8, decay=0.0, step=1, null=False):
    entry = dict(param=4096, grad=8192, exp_avg=16384, exp_avg_sq=32768, exp_avg_scale=None, exp_avg_sq_scale=None, master=None,
                 elements=0)
    table = (_native.AdamwTensor * 1)(_native.AdamwTensor(**{**entry, **(tensor or {})}))
    return _native.load().attnres_hip_adamw(None if null else table, count, param_dtype, grad_dtype, bits, lr, None, beta1, beta2, eps, decay,
                                            step, None, None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(count=-1), _native.ERR_SHAPE), (dict(param_dtype=3), _native.ERR_SHAPE), (dict(param_dtype=0, grad_dtype=1), _native.ERR_SHAPE),
    (dict(bits=16), _native.ERR_SCALAR), (dict(beta1=1.0), _native.ERR_SCALAR), (dict(beta2=float("nan")), _native.ERR_SCALAR),
    (dict(eps=-1.0), _native.ERR_SCALAR), (dict(decay=float("inf")), _native.ERR_SCALAR), (dict(lr=float("nan")), _native.ERR_SCALAR),
    (dict(step=0), _native.ERR_SCALAR), (dict(null=True), _native.ERR_NULL_POINTER), (dict(tensor=dict(elements=-1)), _native.ERR_SHAPE),
    (dict(tensor=dict(elements=4, param=None)), _native.ERR_NULL_POINTER), (dict(tensor=dict(elements=4, grad=None)), _native.ERR_NULL_POINTER),
    (dict(tensor=dict(elements=4), bits=8), _native.ERR_NULL_POINTER), (dict(tensor=dict(elements=4, master=4096)), _native.ERR_SHAPE),
    (dict(tensor=dict(elements=4, param=4098)), _native.ERR_STRIDE), (dict(tensor=dict(elements=4, exp_avg=4097)), _native.ERR_STRIDE),
])
def test_c_abi_refusals(kw, status):
    assert _abi(**kw) == status
    assert _native.load().attnres_hip_last_error()


def test_nothing_to_do():
    assert _abi() == _native.OK  # a tensor without elements
    assert _abi(count=0, null=True) == _native.OK
