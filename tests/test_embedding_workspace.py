"""Sizes of the embedding's workspaces (CPU; nothing launches)."""

from __future__ import annotations

import pytest

from attnres import _native


@pytest.mark.parametrize("batch,length,width,bytes", [
    (0, 5, 64, 0), (64, 1, 64, 0), (65, 1, 64, 2 * 64 * 4), (65536, 1, 64, 1024 * 64 * 4), (2**29, 1, 1, 4096 * 4), (512, 128, 1024, 8 * 128 * 1024 * 4),
    (100, 5000, 64, 0), (5, 0, 64, 0), (2**29 + 1, 1, 1, -1), (4, 4, 8193, -1)])
def test_positions_workspace(batch, length, width, bytes):
    lib = _native.load()
    assert lib.attnres_hip_embedding_positions_workspace_bytes(batch, length, width) == bytes
    whole = lib.attnres_hip_embedding_workspace_bytes(batch, length, 1000, width)
    assert whole == -1 if bytes < 0 else whole >= bytes
