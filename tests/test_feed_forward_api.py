"""The gated feed-forward block's public function and C ABI on the CPU: refusals,
shapes under fake tensors and sizes of what is kept.  Nothing launches."""

from __future__ import annotations

import pytest
import torch

from attnres import _native, layers

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _call(x=torch.zeros(2, 3, 8), gate_up=torch.zeros(20, 8), down=torch.zeros(6, 10), **kw):
    return layers.gated_feed_forward(x, gate_up, down, **kw)


def test_cpu_tensors_are_refused_after_everything_else():
    with pytest.raises(RuntimeError, match="CUDA"):
        _call()


@pytest.mark.parametrize("call,error,match", [
    (lambda: _call([1.0]), TypeError, "x must be a tensor"),
    (lambda: _call(torch.zeros(2, 8, dtype=torch.float64)), TypeError, "bfloat16"),
    (lambda: _call(gate_up=torch.zeros(20, 8, dtype=torch.int64)), TypeError, "gate_up must be one of"),
    (lambda: _call(torch.zeros(())), ValueError, "expected x"),
    (lambda: _call(torch.zeros(2, 7)), ValueError, "expected x"),
    (lambda: _call(gate_up=torch.zeros(8)), ValueError, "gate_up"),
    (lambda: _call(gate_up=torch.zeros(21, 8)), ValueError, "gate_up"),
    (lambda: _call(down=torch.zeros(10, 6)), ValueError, "down"),
    (lambda: _call(down=torch.zeros(10)), ValueError, "down"),
    (lambda: _call(torch.zeros(2, 8193), torch.zeros(20, 8193)), ValueError, "D<=8192"),
    (lambda: _call(torch.zeros(2, 0), torch.zeros(20, 0)), ValueError, "D<=8192"),
    (lambda: _call(down=torch.zeros(8193, 10)), ValueError, "E<=8192"),
    (lambda: _call(down=torch.zeros(0, 10)), ValueError, "E<=8192"),
    (lambda: _call(gate_up=torch.zeros(0, 8), down=torch.zeros(6, 0)), ValueError, "F<=65536"),
    (lambda: _call(gate_up=torch.zeros(1, 8).expand(131074, 8), down=torch.zeros(6, 1).expand(6, 65537)), ValueError, "F<=65536"),
    (lambda: _call(torch.zeros(1, 8).expand(2**24 + 1, 8)), ValueError, "rows"),
    (lambda: _call(torch.zeros(1, 8).expand(2**24, 8), torch.zeros(1, 8).expand(65536, 8), torch.zeros(6, 1).expand(6, 32768)),
     ValueError, "tiles"),
    (lambda: _call(gate_up=torch.zeros(20, 8, dtype=BF16)), TypeError, "dtype of x"),
    (lambda: _call(down=torch.zeros(6, 10, dtype=FP16)), TypeError, "dtype of x"),
    (lambda: _call(down=torch.zeros(6, 10, device="meta")), TypeError, "device"),
    (lambda: _call(activation="relu"), ValueError, "activation"),
    (lambda: _call(activation=0), ValueError, "activation"),
    (lambda: _call(recompute=1), TypeError, "recompute"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, gate_up, down = (torch.empty(s, device="cuda", dtype=BF16) for s in ((2, 3, 40), (160, 40), (24, 80)))
        out, saved = layers._gated_feed_forward(x, gate_up, down, 0, True)
        assert out.shape == (2, 3, 24) and out.dtype == BF16 and saved.dtype == torch.uint8
        grads = layers._gated_feed_forward_backward(out, x, gate_up, down, saved, 0, True, False, True)
        assert [g.shape for g in grads] == [x.shape, torch.Size([0]), down.shape]


@pytest.mark.parametrize("rows,hidden", [(0, 32), (1, 1), (16, 32), (17, 33), (255, 100), (4096, 2816)])
@pytest.mark.parametrize("code,dtype", [(0, BF16), (1, FP16), (2, FP32)])
def test_saved_bytes_of_the_fake_kernel(rows, hidden, code, dtype):
    bytes = _native.load().attnres_hip_gated_ffn_saved_bytes(rows, 64, hidden, 64, code)
    assert bytes == layers._feed_forward_saved_bytes(rows, hidden, dtype)
    if rows % 16 == 0 and hidden % 32 == 0:
        assert bytes == rows * hidden * (8 if dtype == FP32 else 6)


@pytest.mark.parametrize("sizes", [(-1, 8, 8, 8, 0), (2**24 + 1, 8, 8, 8, 0), (4, 0, 8, 8, 0), (4, 8193, 8, 8, 0), (4, 8, 0, 8, 0),
                                   (4, 8, 2**16 + 1, 8, 0), (4, 8, 8, 0, 0), (4, 8, 8, 8193, 0), (4, 8, 8, 8, 3),
                                   (2**24, 8, 2**15, 8, 0)])
def test_sizes_outside_the_envelope(sizes):
    library = _native.load()
    assert library.attnres_hip_gated_ffn_saved_bytes(*sizes) == -1
    assert library.attnres_hip_gated_ffn_workspace_bytes(*sizes, 0) == -1


def _forward(x=4096, x_stride=64, gate_up=4096, gate_up_stride=64, down=4096, down_stride=96, rows=32, width=64, hidden=96,
             out_width=32, dtype=0, activation=0, out=4096, saved=4096, workspace=4096, bytes=1 << 40):
    return _native.load().attnres_hip_gated_ffn_forward(x, x_stride, gate_up, gate_up_stride, down, down_stride, rows, width, hidden,
                                                        out_width, dtype, activation, out, saved, workspace, bytes, None)


def _backward(grad_out=4096, x=4096, x_stride=64, gate_up=4096, gate_up_stride=64, down=4096, down_stride=96, rows=32, width=64,
              hidden=96, out_width=32, dtype=0, activation=0, saved=4096, workspace=4096, bytes=1 << 40):
    return _native.load().attnres_hip_gated_ffn_backward(grad_out, x, x_stride, gate_up, gate_up_stride, down, down_stride, rows, width,
                                                         hidden, out_width, dtype, activation, saved, None, None, None, workspace, bytes,
                                                         None)


_COMMON = [
    (dict(rows=-1), _native.ERR_SHAPE), (dict(rows=2**24 + 1), _native.ERR_SHAPE), (dict(width=0), _native.ERR_SHAPE),
    (dict(out_width=8193), _native.ERR_SHAPE), (dict(hidden=2**16 + 1), _native.ERR_SHAPE), (dict(dtype=3), _native.ERR_SHAPE),
    (dict(activation=2), _native.ERR_SCALAR), (dict(x=None), _native.ERR_NULL_POINTER), (dict(gate_up=None), _native.ERR_NULL_POINTER),
    (dict(down=None), _native.ERR_NULL_POINTER), (dict(x_stride=-8), _native.ERR_STRIDE), (dict(x=4098), _native.ERR_STRIDE),
    (dict(x_stride=65), _native.ERR_STRIDE), (dict(gate_up_stride=56), _native.ERR_STRIDE),
    (dict(gate_up_stride=2**24), _native.ERR_STRIDE), (dict(down=4100), _native.ERR_STRIDE), (dict(down_stride=88), _native.ERR_STRIDE),
    (dict(workspace=None), _native.ERR_WORKSPACE), (dict(workspace=4104), _native.ERR_WORKSPACE), (dict(bytes=0), _native.ERR_WORKSPACE),
    (dict(saved=4104), _native.ERR_WORKSPACE),
]


@pytest.mark.parametrize("call,overrides,status", [(c, o, s) for c in (_forward, _backward) for o, s in _COMMON] + [
    (_forward, dict(out=None), _native.ERR_NULL_POINTER), (_backward, dict(grad_out=None), _native.ERR_NULL_POINTER),
    (_backward, dict(grad_out=4098), _native.ERR_STRIDE), (_backward, dict(rows=0), _native.ERR_SHAPE)])
def test_c_abi_refusals(call, overrides, status):
    assert call(**overrides) == status
    assert _native.load().attnres_hip_last_error()


def test_nothing_to_do():
    assert _forward(rows=0) == _native.OK
    assert _backward() == _native.OK  # no gradient is wanted


def test_workspaces_are_of_the_shape_alone():
    size = _native.load().attnres_hip_gated_ffn_workspace_bytes
    shape = (300, 64, 96, 64)
    forward, backward, again = (size(*shape, 0, p) for p in range(3))
    saved = _native.load().attnres_hip_gated_ffn_saved_bytes(*shape, 0)
    assert 0 < forward < backward and again == backward + -(-saved // 256) * 256
    assert size(*shape, 0, 3) == -1
    for short in (forward - 1, 0):
        assert _forward(rows=300, bytes=short, out_width=64) == _native.ERR_WORKSPACE


@pytest.mark.parametrize("call", [_forward, _backward])
@pytest.mark.parametrize("overrides", [dict(x=4100), dict(x_stride=68), dict(down=4104), dict(gate_up=4104),
                                       dict(hidden=192, gate_up_stride=2**22, down_stride=192)])
def test_fp32_operands_in_place_are_checked(call, overrides):
    assert call(dtype=2, **overrides) == _native.ERR_STRIDE
