"""What the backward of dense attention asks for, without a GPU: its workspace and launches."""
import ctypes

import pytest

from ops_amd import _lib
from tests.test_dense_host import _bwd


def _need(**kw):
    return _lib.load().sfa_dense_bwd_workspace_size(ctypes.byref(_bwd(kw)))


@pytest.mark.parametrize("dtype", [_lib.SFA_DTYPE_F32, _lib.SFA_DTYPE_BF16])
@pytest.mark.parametrize("Dqk,Dv", [(192, 128), (300, 20), (576, 512), (40, 200)])
def test_wide_heads_keep_two_deltas(dtype, Dqk, Dv):
    """A row's dq is several workgroups' there: the delta that they read is not the array that
    one of them writes.  (S such that dk and dv have enough blocks to need no partial sums.)"""
    rows = 2 * 8192 * 16
    need = _need(dtype=dtype, kv_dtype=dtype, S=8192, Hkv=16, Dqk=Dqk, Dv=Dv)
    assert 3 * 4 * rows <= need < 4 * 4 * rows
    assert 2 * 4 * rows <= _need(dtype=dtype, kv_dtype=dtype, S=8192, Hkv=16, Dqk=100, Dv=40) < 3 * 4 * rows
