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


@pytest.mark.parametrize("B,S,Hq,Hkv,D", [(1, 8192, 32, 8, 128), (1, 32768, 64, 8, 128), (2, 5000, 16, 2, 64), (4, 300, 8, 8, 64)])
def test_partial_sums_do_not_grow_with_the_first_tokens(B, S, Hq, Hkv, D):
    """dk and dv of key blocks that many rows see are of several workgroups' partial sums (128
    keys of float32).  Cut into pieces of a share of all rows there are 1024 pieces and one a
    block, five of some 256 blocks that level the last round; the first tokens' no more."""
    blocks = B * Hkv * ((S + 127) // 128)
    rows, part = 2 * 4 * B * S * Hq, 128 * 2 * D * 4
    most = rows + 2 * 512 + (1024 + blocks + 5 * (256 + B * Hkv)) * part + 16 * (blocks + 4096)
    for window in (0, 1, 64, 1024, S - 1, S, (1 << 31) - 1):
        for first in (0, 1, 4, 64, 1000, S // 2, S - 300, S - 100, S - 1, S, S + 1, (1 << 31) - 1):
            first = max(first, 0)
            need = _need(B=B, S=S, Hq=Hq, Hkv=Hkv, Dqk=D, Dv=D, window=window, first=first)
            assert rows <= need <= most, (window, first, need)


def test_masks_that_are_causal():
    """A window or first tokens that reach every row change nothing."""
    for dtype in (_lib.SFA_DTYPE_F32, _lib.SFA_DTYPE_BF16):
        kw = dict(B=1, S=4096, Hq=16, Hkv=2, dtype=dtype, kv_dtype=dtype)
        want = _need(**kw)
        for window, first in ((0, 7), (4096, 0), (4096, 100), (5000, 4096), (3, 4096), (1, (1 << 31) - 1)):
            assert _need(**kw, window=window, first=first) == want, (window, first)
