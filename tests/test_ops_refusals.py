"""Calls of the operators around the attention that the host layer refuses, with
the GPU's checks passed by CPU tensors.  CPU only."""
import ctypes

import pytest
import torch

import ops_amd
from ops_amd import _lib
from tests.host_calls import launches  # noqa: F401


def test_append_without_k_rows(launches):  # noqa: F811
    """No launch would turn q: its memory would be returned as it was allocated."""
    q, k, pool = torch.randn(2, 3, 4, 64), torch.randn(2, 3, 0, 64), torch.randn(9, 16, 0, 64)
    pos, bt = torch.arange(3), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="needs k rows"):
        ops_amd.qk_norm_rope_append(q, k, None, pool, None, bt, pos, pos, ops_amd.rope_frequencies(64))
    empty = ops_amd.qk_norm_rope_append(q[:0], q[:0], None, torch.randn(9, 16, 4, 64), None, bt[:0], pos, pos,
                                        ops_amd.rope_frequencies(64))
    assert empty.shape == (0, 3, 4, 64) and launches == []


@pytest.mark.parametrize("kw", [dict(B=1 << 24, T=1, Hq=1, Hkv=1, Dqk=64, Dv=64), dict(B=1 << 22, T=1, Hq=4, Hkv=4, Dqk=128, Dv=128),
                                dict(B=1 << 21, T=64, Hq=1, Hkv=1, Dqk=77, Dv=33),
                                dict(B=1 << 23, T=1, Hq=1, Hkv=1, Dqk=576, Dv=512)])
def test_tree_of_more_rows_than_a_launch_holds(kw):
    """(2^32 threads; before any HIP call)"""
    from tests.test_ops_host import _pages, _tree
    lib = _lib.load()
    a, pg = _tree(**kw), _pages(max_pages=4096, bt_sb=4096, page_size=64, num_pages=100)
    if kw["Dqk"] == 576:
        a.v = a.k
    assert lib.sfa_tree_fwd(ctypes.byref(a), ctypes.byref(pg), 0x10000, 1 << 40, None) == _lib.SFA_E_UNSUPPORTED
    assert b"launch" in lib.sfa_last_error()
    assert lib.sfa_tree_fwd_workspace_size(ctypes.byref(a), ctypes.byref(pg)) == 0


def test_sizes_that_do_not_fit_the_interface(launches):  # noqa: F811
    """A ValueError as for every other argument, and no size cut to 32 bits."""
    i = torch.zeros(2, dtype=torch.int32)
    bt = torch.zeros(2, 2, dtype=torch.int32)
    for size in (1 << 31, 1 << 40, 1 << 70):
        with pytest.raises(ValueError, match="interface"):
            ops_amd.cache_extend(bt, i, i, i, size)
        with pytest.raises(ValueError, match="interface"):
            ops_amd.cache_free(bt, i, i, i, page_size=size)
    wide = torch.zeros(1, 16, 1, 64).expand((1 << 32) + 1, 16, 1, 64)
    x, pos, mask = torch.zeros(2, 3, 1, 64), torch.arange(3), torch.ones(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="past 2\\^31"):
        ops_amd.tree_attention_paged(x, wide, wide, bt, i, mask)
    with pytest.raises(ValueError, match="expanded"):
        ops_amd.qk_norm_rope_append(None, x, None, wide, None, bt, pos, pos, ops_amd.rope_frequencies(64))
    assert launches == []


def test_forms_without_a_gradient_refuse_inputs_that_want_one(launches):  # noqa: F811
    q, pool, sink = torch.randn(2, 3, 4, 64), torch.randn(9, 16, 2, 64), torch.zeros(4)
    bt, ctx, mask = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.ones(2, 3, dtype=torch.int64)
    pos, freq = torch.arange(3), ops_amd.rope_frequencies(64)

    def leaf(t):
        return t.clone().requires_grad_(True)

    def tree(q=q, k=pool, v=pool, sink=sink):
        return ops_amd.tree_attention_paged(q, k, v, bt, ctx, mask, attn_sink=sink)

    calls = [lambda: tree(q=leaf(q)), lambda: tree(k=leaf(pool)), lambda: tree(v=leaf(pool)), lambda: tree(sink=leaf(sink)),
             lambda: ops_amd.qk_norm_rope_append(leaf(q), q[:, :, :2], q[:, :, :2], pool, pool.clone(), bt, pos, pos, freq),
             lambda: ops_amd.rotary_embedding(leaf(q), pos, freq, out=torch.empty_like(q))]
    for c in calls:
        with pytest.raises(ValueError, match="gradient"):
            c()
    assert launches == []
    tree()
    with torch.no_grad():
        for c in calls:
            c()
    assert len(launches) == 1 + len(calls)


def test_row_counts_past_64_bits():
    """Their product would come back negative and pass for small; before any HIP call."""
    from tests.test_ops_host import _pages, _rope, _tree
    lib, top = _lib.load(), (1 << 31) - 1
    for kw in (dict(B=top, S=top), dict(B=top, S=top, Hq=2, Hkv=1), dict(B=top, S=2, Hq=top, Hkv=top), dict(B=1, S=top, Hq=1, Hkv=1)):
        assert lib.sfa_rope_fwd(ctypes.byref(_rope(**kw)), None, None) == _lib.SFA_E_UNSUPPORTED
        assert lib.sfa_rope_bwd(ctypes.byref(_rope(**kw)), 0x10000, 1 << 40, None) == _lib.SFA_E_UNSUPPORTED
    for kw in (dict(B=top, T=64, Hq=top - 1, Hkv=2), dict(B=top, T=2, Hq=1 << 30, Hkv=1)):
        a, pg = _tree(**kw), _pages(bt_sb=4)
        assert lib.sfa_tree_fwd(ctypes.byref(a), ctypes.byref(pg), 0x10000, 1 << 40, None) == _lib.SFA_E_UNSUPPORTED
