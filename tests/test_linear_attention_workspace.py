"""The C entries of linear attention refuse a workspace off the boundary their stores need.  Sizes
and pointers are checked before anything is launched, so this needs no GPU."""

import ctypes

import pytest

from pytorch_morlet_fdwt_b200 import _lib

from .test_token_ops_host import INVALID, WORKSPACE, _desc


@pytest.mark.parametrize("off", [1, 4, 8, 16, 31])
def test_misaligned_workspace_is_refused(off):
    lib = _lib.load()
    ok = 4096  # a pointer that no call below reaches
    long = _desc(heads=1, kv_heads=1, batch=1, length=1 << 20)  # states between segments
    at = ctypes.addressof(long)
    need = lib.fdwt_linattn_forward_workspace(at)
    assert need > 0
    assert lib.fdwt_linattn_forward(at, *[ok] * 8, ok + off, need, None) == INVALID
    assert lib.fdwt_linattn_forward(at, *[ok] * 8, ok + off, need - 1, None) == WORKSPACE
    shared = _desc(heads=4, kv_heads=1)  # gradients of each head
    at = ctypes.addressof(shared)
    need = lib.fdwt_linattn_backward_workspace(at)
    assert lib.fdwt_linattn_backward(at, *[ok] * 12, ok + off, need, None) == INVALID
