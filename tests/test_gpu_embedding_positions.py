"""The positions' gradient of an embedding over large batches: a sum of many rows, which one FP32 accumulator does not hold."""

from __future__ import annotations

import pytest
import torch

from attnres import _native, layers
from layer_reference import U32, assert_within

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _positions_gradient(tokens, rows, width, grad, dtype, table_rows=7, want_table=True):
    weight = torch.zeros(table_rows, width, device="cuda", dtype=FP32, requires_grad=want_table)
    positions = torch.zeros(rows, width, device="cuda", dtype=FP32, requires_grad=True)
    out = layers.embedding(tokens, weight, positions, dtype=dtype)
    leaves = (positions, weight) if want_table else (positions,)
    return torch.autograd.grad(out, leaves, grad)


@pytest.mark.parametrize("batch,length,width", [(65536, 1, 64), (4096, 16, 256), (512, 128, 1000), (20000, 3, 8), (1000, 7, 2049),
                                                (33, 40, 72), (129, 1, 1), (64, 5, 24), (65, 5, 24)])
@pytest.mark.parametrize("want_table", [False, True])
def test_sums_over_large_batches(batch, length, width, want_table):
    """Equal values of one sign, whose roundings all go one way in a long sum.  At most 64 additions in a row within a block of
    rows, batch / 64 / parts of blocks (of these sizes at most 64), a few hundred partial sums: 512 roundings in a row in all."""
    g = torch.Generator(device="cuda").manual_seed(batch + length)
    tokens = torch.randint(7, (batch, length), generator=g, device="cuda", dtype=torch.int32)
    grad = torch.full((batch, length, width), 0.1, device="cuda")
    grad[:, :, width // 2:] = torch.randn(batch, length, width - width // 2, generator=g, device="cuda")
    got = _positions_gradient(tokens, length + 3, width, grad, FP32, want_table=want_table)
    expected = torch.zeros(length + 3, width, device="cuda", dtype=torch.float64)
    size = torch.zeros_like(expected)
    expected[:length], size[:length] = grad.double().sum(0), grad.double().abs().sum(0)
    assert_within("dpos", got[0], expected, 512 * U32 * size)
    again = _positions_gradient(tokens, length + 3, width, grad, FP32, want_table=want_table)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("batch,length,width", [(65536, 1, 64), (3000, 6, 300), (65, 5, 24)])
def test_sums_through_the_c_abi_with_and_without_a_workspace(batch, length, width):
    """Without one the blocks of 64 are added up in one sum: batch / 64 + 64 roundings in a row."""
    lib = _native.load()
    g = torch.Generator(device="cuda").manual_seed(batch)
    grad = torch.rand(batch, length, width, generator=g, device="cuda")
    tokens = torch.zeros(batch, length, device="cuda", dtype=torch.int64)
    size = lib.attnres_hip_embedding_positions_workspace_bytes(batch, length, width)
    workspace = torch.empty(size, device="cuda", dtype=torch.uint8)
    expected = torch.zeros(length + 2, width, device="cuda", dtype=torch.float64)
    expected[:length] = grad.double().sum(0)
    for pointer, bytes in ((None, 0), (workspace.data_ptr(), size), (workspace.data_ptr(), max(size - 1, 0))):
        out = torch.full((length + 2, width), 7.0, device="cuda")
        status = lib.attnres_hip_embedding_backward(grad.data_ptr(), 2, tokens.data_ptr(), 8, batch, length, 10, width, 2, 1.0, None,
                                                    out.data_ptr(), length + 2, pointer, bytes, torch.cuda.current_stream().cuda_stream)
        assert status == 0, lib.attnres_hip_last_error().decode()
        assert_within("dpos", out, expected, (batch / 64 + 64) * U32 * expected)


def test_a_batch_beyond_what_an_accumulator_counts():
    """2^24 + 2^20 ones: a running FP32 sum of ones ends at 2^24."""
    batch = 2**24 + 2**20
    tokens = torch.zeros(batch, 1, device="cuda", dtype=torch.int32)
    (got,) = _positions_gradient(tokens, 1, 1, torch.ones(batch, 1, 1, device="cuda", dtype=BF16), BF16, want_table=False)
    assert float(got[0, 0]) == float(batch)
