"""Workspace sizes of the group norm, on the CPU: in proportion to the tensors, at any width."""
from __future__ import annotations

import pytest

from bysj_amd.kernels import _lib

pytestmark = pytest.mark.skipif(not _lib.LIBRARY_PATH.exists(), reason="libdpa4k.so is not built")


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("channels,groups", [(4095, 4095), (4095, 819), (4096, 4096), (2047, 2047), (64, 64), (63, 63), (4093, 1)])
@pytest.mark.parametrize("samples,rows", [(1, 1 << 10), (1, 1 << 12), (1, 1 << 20), (1000, 1 << 14), (1 << 12, 1 << 12)])
def test_workspaces_stay_in_proportion(samples, rows, channels, groups, backward):
    """A (piece, group) has a slot of 12 bytes at most and a (tile, channel) a pair of sums; of pieces there are a sample's
    and a tile's, and a tile is 16 KB at least or one row: with 24 bytes to a channel of either kind all fits."""
    lib = _lib.load()
    for kind, size in ((_lib.TYPE_F32, 4), (_lib.TYPE_BF16, 2)):
        nbytes = lib.dpa4k_group_norm_workspace_size(samples, rows, 1, channels, groups, 1, -1, kind, backward)
        tiles = min(rows, rows * channels * size // 8192 + 1)
        assert 0 < nbytes <= 24 * channels * (samples + tiles) + 4096
