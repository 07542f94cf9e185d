"""Sizes at the C entry points of the optimiser that no memory holds, on the CPU: refused before any device call."""
from __future__ import annotations

import ctypes

import pytest

from bysj_amd.kernels import _lib

pytestmark = pytest.mark.skipif(not _lib.LIBRARY_PATH.exists(), reason="libdpa4k.so is not built")


def test_gradient_lists_are_checked_whole_before_the_first_launch():
    """180 gradients make a launch; the 181st is too large, and the workspace of such a list is 0 bytes."""
    lib, n = _lib.load(), 181
    pointers, types = (ctypes.c_void_p * n)(*[256] * n), (ctypes.c_int32 * n)()    # never dereferenced
    counts = (ctypes.c_int64 * n)(*[4] * 180, 1 << 44)
    some = ctypes.c_void_p(256)
    assert lib.dpa4k_grad_norm_workspace_size(counts, n) == 0
    for workspace, nbytes in ((None, 0), (some, 1 << 20)):
        assert lib.dpa4k_grad_norm(pointers, counts, types, n, 1.0, some, some, workspace, nbytes, None) == _lib.EINVAL
        assert "too many" in lib.dpa4k_last_error().decode()
