"""Operators around the attention, without a GPU: argument structs against the
header, refusals of the C entry points (before any HIP call) and of the host
layer, and the rotation's frequencies."""
import ctypes
import math
import subprocess

import pytest
import torch

import ops_amd
from ops_amd import _lib
from tests.test_abi import HEADER


def test_struct_layouts_match_header(tmp_path):
    pairs = [("sfa_rope_args", _lib.RopeArgs), ("sfa_tree_args", _lib.TreeArgs), ("sfa_cache_pool", _lib.CachePool),
             ("sfa_cache", _lib.Cache)]
    src = tmp_path / "layout.c"
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    want = []
    for name, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(cls, f).offset)
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-o", str(exe), str(src)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == want


P = 0x10000  # never read: the calls fail before any HIP call


def _rope(**kw):
    a = _lib.RopeArgs()
    a.dtype = a.w_dtype = _lib.SFA_DTYPE_BF16
    a.B, a.S, a.D, a.Hq, a.Hkv, a.rotary_dim, a.q_norm, a.k_norm = 1, 2, 128, 4, 2, 64, 128, 128
    a.eps, a.rope_scale = 1e-6, 1.0
    for n in ("positions", "inv_freq", "q", "k", "q_weight", "k_weight", "q_out", "k_out", "dq", "dk", "dq_weight", "dk_weight"):
        setattr(a, n, P)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def _pages(**kw):
    pg = _lib.KvPages()
    pg.block_table, pg.bt_sb, pg.max_pages, pg.page_size, pg.num_pages = P, 4, 4, 16, 10
    for n, v in kw.items():
        setattr(pg, n, v)
    return pg


@pytest.mark.parametrize("kw", [
    dict(dtype=2), dict(w_dtype=7), dict(dtype=0, w_dtype=1), dict(B=0), dict(S=-1), dict(D=0), dict(D=1025), dict(Hq=0, Hkv=0),
    dict(rotary_dim=63), dict(rotary_dim=130), dict(rope_offset=-2), dict(rope_offset=66), dict(q_norm=129), dict(k_norm=-1),
    dict(eps=-1.0), dict(eps=math.nan), dict(rope_scale=math.inf), dict(positions=None), dict(inv_freq=None), dict(q=None),
    dict(k_out=None), dict(q_weight=None), dict(flags=1)])
def test_rope_refusals(kw):
    lib = _lib.load()
    assert lib.sfa_rope_fwd(ctypes.byref(_rope(**kw)), None, None) == _lib.SFA_E_INVALID
    assert lib.sfa_last_error()


def test_rope_backward_and_append_refusals():
    lib = _lib.load()
    for kw in (dict(dq=None), dict(dk_weight=None), dict(q=None)):
        assert lib.sfa_rope_bwd(ctypes.byref(_rope(**kw)), P, 1 << 30, None) == _lib.SFA_E_INVALID
    need = lib.sfa_rope_bwd_workspace_size(ctypes.byref(_rope()))
    assert need > 0 and lib.sfa_rope_bwd_workspace_size(ctypes.byref(_rope(q_norm=0, k_norm=0))) == 0
    assert lib.sfa_rope_bwd(ctypes.byref(_rope()), P, need - 1, None) == _lib.SFA_E_WORKSPACE
    assert lib.sfa_rope_bwd(ctypes.byref(_rope()), None, need, None) == _lib.SFA_E_WORKSPACE
    for kw, pk in ((dict(), {}), (dict(slots=P, Dv=8), {}), (dict(slots=P, Dv=-1), {}), (dict(slots=P), dict(page_size=24)),
                   (dict(slots=P), dict(block_table=None)), (dict(slots=P), dict(num_pages=1 << 28)),
                   (dict(slots=P, B=2), dict(bt_sb=3)), (dict(slots=P), dict(flags=1))):
        assert lib.sfa_rope_fwd(ctypes.byref(_rope(**kw)), ctypes.byref(_pages(**pk)), None) == _lib.SFA_E_INVALID
    assert lib.sfa_rope_fwd(ctypes.byref(_rope(B=1 << 16, S=1 << 16)), None, None) == _lib.SFA_E_UNSUPPORTED
    assert lib.sfa_rope_fwd(None, None, None) == _lib.SFA_E_INVALID


def _tree(**kw):
    a = _lib.TreeArgs()
    a.dtype = _lib.SFA_DTYPE_BF16
    a.B, a.T, a.Hq, a.Hkv, a.Dqk, a.Dv, a.scale = 2, 8, 16, 2, 128, 128, 0.1
    for n in ("q", "k", "v", "ctx_lens", "tree_mask", "out", "lse"):
        setattr(a, n, P)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(dtype=2), dict(B=0), dict(T=0), dict(T=65), dict(Hq=15), dict(Hkv=0), dict(Dqk=0), dict(Dv=1025), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(q=None), dict(tree_mask=None), dict(lse=None),
    dict(flags=4)])
def test_tree_refusals(kw):
    lib = _lib.load()
    a, pg = _tree(**kw), _pages()
    assert lib.sfa_tree_fwd_workspace_size(ctypes.byref(a), ctypes.byref(pg)) == 0
    assert lib.sfa_tree_fwd(ctypes.byref(a), ctypes.byref(pg), P, 1 << 30, None) == _lib.SFA_E_INVALID


def test_tree_pages_and_workspace():
    lib = _lib.load()
    for pk in (dict(page_size=0), dict(max_pages=0), dict(num_pages=0), dict(block_table=None), dict(bt_sb=1),
               dict(max_pages=1 << 28, bt_sb=1 << 28)):
        assert lib.sfa_tree_fwd(ctypes.byref(_tree()), ctypes.byref(_pages(**pk)), P, 1 << 30, None) == _lib.SFA_E_INVALID
    pg = _pages(max_pages=2048, bt_sb=2048, page_size=64, num_pages=5000)
    need = lib.sfa_tree_fwd_workspace_size(ctypes.byref(_tree()), ctypes.byref(pg))
    assert need > 0
    assert lib.sfa_tree_fwd(ctypes.byref(_tree()), ctypes.byref(pg), P, need - 1, None) == _lib.SFA_E_WORKSPACE
    assert lib.sfa_tree_fwd(ctypes.byref(_tree()), ctypes.byref(pg), None, need, None) == _lib.SFA_E_WORKSPACE


def _cache(**kw):
    pools = (_lib.CachePool * 2)()
    for q in pools:
        q.base, q.page_stride, q.page_bytes = P, 4096, 4096
    c = _lib.Cache()
    c.pools, c.npools, c.B, c.max_pages, c.page_size, c.num_pages = ctypes.addressof(pools), 2, 4, 8, 16, 100
    c.block_table, c.bt_sb, c.ref_counts, c.kv_lens = P, 8, P, P
    for n, v in kw.items():
        if n in ("page_stride", "page_bytes", "base"):
            setattr(pools[1], n, v)
        else:
            setattr(c, n, v)
    c._keep = pools
    return c


@pytest.mark.parametrize("kw", [
    dict(page_size=12), dict(page_size=0), dict(num_pages=0), dict(num_pages=1 << 28), dict(flags=1), dict(npools=0),
    dict(npools=5000), dict(pools=None), dict(page_bytes=4090), dict(page_bytes=0), dict(page_stride=100), dict(base=None),
    dict(block_table=None), dict(B=0), dict(max_pages=0), dict(bt_sb=7), dict(ref_counts=None)])
def test_cache_refusals(kw):
    lib = _lib.load()
    c = ctypes.byref(_cache(**kw))
    assert lib.sfa_cache_compact(c, P, P, 1 << 30, None) == _lib.SFA_E_INVALID
    assert lib.sfa_last_error()


def test_cache_call_refusals():
    lib = _lib.load()
    c = ctypes.byref(_cache())
    need = lib.sfa_cache_workspace_size(c, 5)
    assert lib.sfa_cache_copy(c, P, P, 5, P, need - 1, None) == _lib.SFA_E_WORKSPACE
    assert lib.sfa_cache_copy(c, P, None, 5, P, need, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_copy(c, P, P, -1, P, need, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_copy(c, P, P, 0, None, 0, None) == _lib.SFA_OK
    assert lib.sfa_cache_fork(c, P, P, 5, None, P, need, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_fork(c, P, P, 70000, P, P, 1 << 30, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_fork(ctypes.byref(_cache(kv_lens=None)), P, P, 5, P, P, need, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_fork(ctypes.byref(_cache(B=9000)), P, P, 5, P, P, need, None) == _lib.SFA_E_UNSUPPORTED
    assert lib.sfa_cache_extend(ctypes.byref(_cache(B=9000)), P, P, P, need, None) == _lib.SFA_E_UNSUPPORTED
    assert lib.sfa_cache_extend(c, None, P, P, need, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_free(c, None, None, 3, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_free(c, P, None, 70000, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_keep_path(c, P, P, 4, 65, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_keep_path(c, None, P, 4, 4, None) == _lib.SFA_E_INVALID
    assert lib.sfa_cache_workspace_size(c, -1) == 0


def test_host_layer_refuses_cpu_tensors_and_bad_shapes():
    x, pos, f = torch.zeros(1, 2, 4, 64), torch.zeros(1, 2, dtype=torch.int32), ops_amd.rope_frequencies(64)
    i = torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros(4, 16, 2, 64)
    calls = [
        lambda: ops_amd.rotary_embedding(x, pos, f),
        lambda: ops_amd.rotary_embedding(x[0], pos, f),
        lambda: ops_amd.qk_norm_rope(x, x, pos, f),
        lambda: ops_amd.qk_norm_rope_append(x, x, x, pool, pool, i.view(1, 1), pos, pos, f),
        lambda: ops_amd.tree_attention_paged(x, pool, pool, i.view(1, 1), i, torch.zeros(1, 2, dtype=torch.int64)),
        lambda: ops_amd.tree_attention_paged(x[0], pool, pool, i.view(1, 1), i, torch.zeros(1, 2, dtype=torch.int64)),
        lambda: ops_amd.cache_copy_pages([pool], i, i),
        lambda: ops_amd.cache_copy_pages([], i, i),
        lambda: ops_amd.cache_fork(i.view(1, 1), i, i, i, i, [pool]),
        lambda: ops_amd.cache_free(i.view(1, 1), i, i),
        lambda: ops_amd.cache_extend(i.view(1, 1), i, i, i, 16),
        lambda: ops_amd.cache_compact(i.view(1, 1), i, [pool]),
        lambda: ops_amd.cache_keep_path([pool], i.view(1, 1), i, i.view(1, 1)),
    ]
    for c in calls:
        with pytest.raises(ValueError):
            c()


def test_rope_frequencies():
    f = ops_amd.rope_frequencies(8, theta=100.0)
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-14)
    assert torch.equal(ops_amd.rope_frequencies(8, theta=100.0, scaling="linear", factor=4.0), f / 4)
    n = ops_amd.rope_frequencies(64, scaling="ntk", factor=8.0)
    p = ops_amd.rope_frequencies(64)
    assert float(n[0]) == 1.0 and abs(float(n[-1] * 8 / p[-1]) - 1) < 1e-12
    y = ops_amd.rope_frequencies(64, scaling="yarn", factor=16.0, original_length=4096)
    turns = 4096 * p / (2 * math.pi)
    assert torch.equal(y[turns > 64], p[turns > 64]) and torch.allclose(y[turns < 0.5], p[turns < 0.5] / 16, rtol=1e-14)
    assert bool(((y <= p) & (y >= p / 16 - 1e-18)).all())
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, theta=1.0), dict(rotary_dim=8, factor=0.0),
                dict(rotary_dim=8, scaling="other"), dict(rotary_dim=2, scaling="ntk"), dict(rotary_dim=8, scaling="yarn")):
        with pytest.raises(ValueError):
            ops_amd.rope_frequencies(**bad)


def test_sizes_past_the_counters_are_refused():
    lib = _lib.load()
    one = dict(num_pages=(1 << 30) + 1, page_size=1, npools=0)
    assert lib.sfa_cache_free(ctypes.byref(_cache(**one)), P, None, 1, None) == _lib.SFA_E_UNSUPPORTED
    many = dict(B=1 << 12, max_pages=1 << 20, bt_sb=1 << 20)
    assert lib.sfa_cache_extend(ctypes.byref(_cache(**many)), P, P, P, 1 << 30, None) == _lib.SFA_E_UNSUPPORTED


def test_tensors_that_are_written():
    from ops_amd._host import written
    t = torch.zeros(3, 4)
    v = t._version
    written(t, None, t[:1].expand(1, 4), t[:0].expand(0, 4))
    assert t._version > v
    with pytest.raises(ValueError, match="expanded"):
        written(t[:1].expand(3, 4))
    w = t.clone().requires_grad_(True)
    with pytest.raises(ValueError, match="gradient"):
        written(w)
    with torch.no_grad():
        written(w)
    with torch.inference_mode():
        written(torch.zeros(2))
