"""AdamW steps that write 128 MB and more, which go past the caches: against the definition in FP64, and bit for bit against the
same tensors in calls of their own, which do not (an element's result depends on no other tensor)."""

from __future__ import annotations

import pytest
import torch

from attnres import optim
from test_gpu_adamw import BF16, FP16, FP32, OPTIONS, _check, _copy, _inputs

pytestmark = pytest.mark.gpu

PAST_CACHES = 128 * 2**20


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def _written(state):
    """Bytes that a step writes, per tensor, without scales."""
    size = state["exp_avgs"][0].element_size()
    return [p.numel() * (p.element_size() + 2 * size + (0 if state["masters"] is None else 4)) for p in state["params"]]


def _shifted(t):
    """At the third element of a buffer."""
    return torch.empty(t.numel() + 3, dtype=t.dtype, device="cuda")[3:].view(t.shape).copy_(t)


# dtype, gradients' dtype, masters, bits, elements of the larger tensors
KINDS = [(FP32, FP32, False, 32, 5_000_001), (FP32, FP32, False, 8, 9_000_001), (BF16, BF16, True, 32, 4_300_001), (FP16, FP32, True, 8, 8_000_001),
         (BF16, BF16, False, 8, 15_000_001), (FP16, FP16, False, 32, 6_000_001)]


@pytest.mark.parametrize("dtype,grad_dtype,masters,bits,elements", KINDS)
def test_large_steps(dtype, grad_dtype, masters, bits, elements):
    """Tensors that end inside a lane, a block and a workgroup, one of them at an odd element, and more of them than a launch
    takes."""
    shapes = [(elements,), (1,), (elements // 1537, 1537), (257,), *[(97 * k + 1,) for k in range(60)], (elements + 254,), (4095,)]
    state = _inputs(71, shapes, dtype, grad_dtype, bits, masters)
    for tensors in state.values():
        if tensors is not None:
            tensors[2] = _shifted(tensors[2])
    assert sum(_written(state)) >= PAST_CACHES > max(_written(state))
    alone = _copy(state)
    scale = torch.tensor(0.3, device="cuda")
    _check(state, grad_scale=scale)
    for i in range(len(shapes)):
        one = {k: None if v is None else v[i:i + 1] for k, v in alone.items()}
        optim.adamw_step(**one, grad_scale=scale, **OPTIONS)
    for k, tensors in state.items():
        for i, (a, b) in enumerate(zip(tensors or [], alone[k] or [])):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), (k, i)
