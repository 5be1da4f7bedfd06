"""Dense attention, 8-bit appends and cache reads without a GPU: argument structs
against the header, refusals of the C entry points (before any HIP call) and of
the host layer, and what a call holds until its launch."""
import ctypes
import math
import subprocess

import pytest
import torch

import ops_amd
from ops_amd import _host, _lib, cache, dense, rope
from tests.host_calls import Library, addresses, live
from tests.test_abi import HEADER
from tests.test_ops_host import P, _pages, _rope

F8 = torch.float8_e4m3fn
I32 = torch.int32


def test_struct_layouts_match_header(tmp_path):
    pairs = [("sfa_dense_args", _lib.DenseArgs), ("sfa_dense_bwd_args", _lib.DenseBwdArgs), ("sfa_kv_scales", _lib.KvScales),
             ("sfa_cache_read_args", _lib.CacheReadArgs)]
    src, want = tmp_path / "layout.c", []
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    for name, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(cls, f).offset)
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-o", str(tmp_path / "layout"), str(src)], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == want


def _dense(**kw):
    a = _lib.DenseArgs()
    a.dtype = a.kv_dtype = _lib.SFA_DTYPE_BF16
    a.B, a.S, a.Hq, a.Hkv, a.Dqk, a.Dv, a.scale = 2, 8, 16, 2, 128, 128, 0.1
    for n in ("q", "k", "v", "ctx_lens", "out", "lse"):
        setattr(a, n, P)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def _bwd(fwd=None, **kw):
    a = _lib.DenseBwdArgs()
    a.fwd = _dense(**dict(dict(ctx_lens=None), **(fwd or {})))
    for n in ("dout", "dq", "dk", "dv"):
        setattr(a, n, P)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


BAD = [dict(dtype=2), dict(kv_dtype=0), dict(kv_dtype=2), dict(B=0), dict(S=0), dict(Hq=15), dict(Hkv=0), dict(Dqk=0),
       dict(Dv=1025), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(q=None), dict(out=None),
       dict(lse=None), dict(flags=4), dict(window=-1), dict(first=-1)]


@pytest.mark.parametrize("kw", BAD + [dict(ctx_lens=None)])
def test_dense_refusals(kw):
    lib = _lib.load()
    a, pg = ctypes.byref(_dense(**kw)), ctypes.byref(_pages())
    assert lib.sfa_dense_fwd_workspace_size(a, pg) == 0
    assert lib.sfa_dense_fwd(a, pg, P, 1 << 40, None) == _lib.SFA_E_INVALID
    assert lib.sfa_last_error()


@pytest.mark.parametrize("kw", BAD + [dict(ctx_lens=P)])
def test_dense_backward_refusals(kw):
    lib = _lib.load()
    a = ctypes.byref(_bwd(kw))
    assert lib.sfa_dense_bwd_workspace_size(a) == 0
    assert lib.sfa_dense_bwd(a, P, 1 << 40, None) == _lib.SFA_E_INVALID


def test_dense_pages_workspaces_and_sizes():
    lib, top = _lib.load(), (1 << 31) - 1
    for pk in (dict(page_size=0), dict(max_pages=0), dict(num_pages=0), dict(block_table=None), dict(bt_sb=1),
               dict(max_pages=1 << 28, bt_sb=1 << 28)):
        assert lib.sfa_dense_fwd(ctypes.byref(_dense()), ctypes.byref(_pages(**pk)), P, 1 << 40, None) == _lib.SFA_E_INVALID
    wide = _pages(max_pages=1 << 24, bt_sb=1 << 24, page_size=64)
    assert lib.sfa_dense_fwd(ctypes.byref(_dense()), ctypes.byref(wide), P, 1 << 40, None) == _lib.SFA_E_UNSUPPORTED
    pg = _pages(max_pages=2048, bt_sb=2048, page_size=64, num_pages=5000)
    one = _dense(S=1)
    need = lib.sfa_dense_fwd_workspace_size(ctypes.byref(one), ctypes.byref(pg))
    assert need > 0
    for ws, n in ((P, need - 1), (None, need)):
        assert lib.sfa_dense_fwd(ctypes.byref(one), ctypes.byref(pg), ws, n, None) == _lib.SFA_E_WORKSPACE
    need = lib.sfa_dense_bwd_workspace_size(ctypes.byref(_bwd()))
    assert need >= 2 * 4 * 2 * 8 * 16
    for ws, n in ((P, need - 1), (None, need)):
        assert lib.sfa_dense_bwd(ctypes.byref(_bwd()), ws, n, None) == _lib.SFA_E_WORKSPACE
    for kw in (dict(dout=None), dict(dk=None), dict(flags=1), dict(dsink=P)):
        assert lib.sfa_dense_bwd(ctypes.byref(_bwd(**kw)), P, 1 << 40, None) == _lib.SFA_E_INVALID
    for kw in (dict(B=top, S=64, Hq=top - 1, Hkv=2), dict(B=top, S=2, Hq=1 << 30, Hkv=1), dict(B=1, S=top, Hq=1, Hkv=1),
               dict(B=1 << 25, S=1, Hq=8, Hkv=8)):
        assert lib.sfa_dense_fwd(ctypes.byref(_dense(**kw)), ctypes.byref(pg), P, 1 << 60, None) == _lib.SFA_E_UNSUPPORTED, kw
        assert lib.sfa_dense_bwd(ctypes.byref(_bwd(kw)), P, 1 << 60, None) == _lib.SFA_E_UNSUPPORTED, kw
    assert lib.sfa_dense_fwd(ctypes.byref(_dense(S=(1 << 29) + 1, Hq=1, Hkv=1, B=1, ctx_lens=None)), None, P, 1 << 60,
                             None) == _lib.SFA_E_UNSUPPORTED
    assert lib.sfa_dense_fwd(None, None, P, 1, None) == lib.sfa_dense_bwd(None, P, 1, None) == _lib.SFA_E_INVALID


def test_append_fp8_and_read_refusals():
    lib = _lib.load()
    sc = _lib.KvScales(P, 32, 2, 1, P, 32, 2, 1)
    none = _lib.KvScales()
    a, pg = _rope(slots=P), _pages()
    for args in ((a, pg, none), (_rope(slots=P, Hkv=0), pg, sc), (_rope(), pg, sc), (a, _pages(page_size=24), sc),
                 (_rope(slots=P, Dv=128, v=P, v_out=P), pg, _lib.KvScales(P, 32, 2, 1))):
        assert lib.sfa_rope_append_fp8(*(ctypes.byref(x) for x in args), None) == _lib.SFA_E_INVALID
    assert lib.sfa_rope_append_fp8(ctypes.byref(a), None, ctypes.byref(sc), None) == _lib.SFA_E_INVALID
    assert lib.sfa_rope_append_fp8(ctypes.byref(a), ctypes.byref(pg), None, None) == _lib.SFA_E_INVALID

    def read(**kw):
        r = _lib.CacheReadArgs()
        r.dtype, r.cache_dtype, r.B, r.N, r.H, r.D = 1, 1, 1, 4, 2, 64
        r.cache = r.lens = r.out = P
        for n, v in kw.items():
            setattr(r, n, v)
        return lib.sfa_cache_read(ctypes.byref(r), ctypes.byref(pg), None)
    for kw in (dict(dtype=2), dict(cache_dtype=3), dict(cache_dtype=2), dict(B=0), dict(N=0), dict(D=0), dict(cache=None),
               dict(lens=None), dict(out=None), dict(flags=1)):
        assert read(**kw) == _lib.SFA_E_INVALID, kw
    for kw in (dict(B=1 << 16), dict(N=1 << 26), dict(H=1 << 20, D=1 << 20)):
        if "B" in kw:
            pg.bt_sb = 4
        assert read(**kw) == _lib.SFA_E_UNSUPPORTED, kw


@pytest.fixture
def launches(monkeypatch):
    seen = []
    for m in (_host, dense, cache, rope):
        monkeypatch.setattr(m, "need_gpu", lambda name, t, device=None: None)
        if m is not _host:
            monkeypatch.setattr(m, "call", lambda device, fn, *args: seen.append(
                (fn, args, [n for n, at in addresses(args) if not live(at)])))
    monkeypatch.setattr(_lib, "load", Library)
    return seen


def _rows(h, d=64, grad=False):
    """[2, 3, h, d] with a feature stride other than 1."""
    return torch.randn(2, 3, d, h).transpose(2, 3).requires_grad_(grad)


def _i(*x):
    return torch.tensor(x, dtype=torch.int64)


def test_everything_lives_until_the_launch(launches):
    kc, vc = torch.randn(9, 16, 2, 64), torch.randn(9, 16, 2, 64)
    bt, ctx = _i(0, 1, 2, 3).view(2, 2), _i(3, 4)
    sink = torch.zeros(4, dtype=torch.float64, requires_grad=True)
    with torch.no_grad():
        ops_amd.chunk_attention_paged(_rows(4), kc, vc, bt, ctx, ctx, attn_sink=sink)
        k8, s8 = kc.to(F8), torch.zeros(9, 16, 2, dtype=torch.uint8)
        ops_amd.chunk_attention_paged(_rows(4), k8, k8, bt, ctx, ctx, k_scales=s8, v_scales=s8.transpose(0, 1).contiguous().transpose(0, 1))
        pos, freq = torch.arange(3), ops_amd.rope_frequencies(64).float()
        ops_amd.qk_norm_rope_append(_rows(4), _rows(2), _rows(2), k8, k8.clone(), bt, pos, pos, freq, k_scales=s8, v_scales=s8.clone())
    ops_amd.cache_read(kc, bt, ctx, 5, _i(1, 2))
    out, lse = ops_amd.window_attention(_rows(4, grad=True), _rows(2, grad=True), _rows(2, grad=True), 5, 1, lens=ctx, attn_sink=sink)
    torch.autograd.backward([out, lse], [_rows(4), torch.randn(4, 3, 2).permute(2, 1, 0).double().float()])
    assert [fn for fn, _, _ in launches] == ["sfa_dense_fwd", "sfa_dense_fwd", "sfa_rope_append_fp8", "sfa_cache_read", "sfa_dense_fwd",
                                             "sfa_dense_bwd"]
    assert [(fn, lost) for fn, _, lost in launches if lost] == []
    assert sink.grad.dtype == torch.float64 and sink.grad.shape == (4,)


def test_refusals_of_the_host_layer(launches):
    q, kc = torch.randn(2, 3, 4, 64), torch.randn(9, 16, 2, 64)
    bt, ctx = torch.zeros(2, 2, dtype=I32), torch.zeros(2, dtype=I32)
    k8, s8 = kc.to(F8), torch.zeros(9, 16, 2, dtype=torch.uint8)
    pos, freq = torch.arange(3), ops_amd.rope_frequencies(64)
    leaf = q.clone().requires_grad_(True)

    def chunk(q=q, k=kc, v=kc, bt=bt, ctx=ctx, n=None, **kw):
        return ops_amd.chunk_attention_paged(q, k, v, bt, ctx, n, **kw)

    def app(k=k8, v=None, x=q[:, :, :2], **kw):
        return ops_amd.qk_norm_rope_append(None, x, None if v is None else x, k, v, bt, pos, pos, freq, **kw)

    def win(q=q, k=q[:, :, :2], v=q[:, :, :2], **kw):
        return ops_amd.window_attention(q, k, v, **kw)

    calls = [
        lambda: chunk(q=q[0]), lambda: chunk(q=q.half()), lambda: chunk(q=leaf), lambda: chunk(k=kc.half(), v=kc.half()),
        lambda: chunk(k=k8, v=k8), lambda: chunk(k=k8, v=kc, k_scales=s8, v_scales=s8), lambda: chunk(k_scales=s8),
        lambda: chunk(k=k8, v=k8.clone(), k_scales=s8), lambda: chunk(k=k8, v=k8, k_scales=s8.float()),
        lambda: chunk(k=k8, v=k8, k_scales=s8[1:]), lambda: chunk(v=kc[:, :8]), lambda: chunk(k=kc[:, :15], v=kc[:, :15]),
        lambda: chunk(q=q[..., :32]), lambda: chunk(ctx=ctx[:1]), lambda: chunk(ctx=ctx.float()), lambda: chunk(n=ctx[:1]),
        lambda: chunk(bt=bt[:1]), lambda: chunk(window=0), lambda: chunk(window=-3), lambda: chunk(window=1 << 31),
        lambda: chunk(window=2.5), lambda: chunk(first=-1), lambda: chunk(attn_sink=torch.zeros(3)),
        lambda: chunk(attn_sink=torch.zeros(4, dtype=I32)), lambda: chunk(out=q[..., :32]), lambda: chunk(out=q.bfloat16()),
        lambda: chunk(lse=torch.zeros(2, 3, 3)), lambda: chunk(out=torch.zeros(1, 1, 4, 64).expand(2, 3, 4, 64)),
        lambda: chunk(out=leaf), lambda: chunk(k=kc.transpose(2, 3), v=kc.transpose(2, 3)),
        lambda: app(), lambda: app(k_scales=s8[:, :8]), lambda: app(k=kc, k_scales=s8), lambda: app(k_scales=s8, v=kc),
        lambda: app(k_scales=s8, v=k8.clone()), lambda: app(k_scales=s8, v_scales=s8), lambda: app(k_scales=s8.int()),
        lambda: app(k=k8[..., :32], k_scales=s8), lambda: app(k_scales=s8[..., :1].expand(9, 16, 2)),
        lambda: win(q=q[0]), lambda: win(q=q.half(), k=q.half(), v=q.half()), lambda: win(k=q[:, :, :3]), lambda: win(k=q[:, :2, :2]),
        lambda: win(k=q[:, :, :2].bfloat16()), lambda: win(v=q[:1, :, :2]), lambda: win(k=q[..., :32]), lambda: win(window=0),
        lambda: win(first=-1), lambda: win(lens=ctx[:1]), lambda: win(lens=ctx.bool()), lambda: win(attn_sink=torch.zeros(2)),
        lambda: win(k=q[:, :, :0], v=q[:, :, :0]),
        lambda: ops_amd.cache_read(kc, bt, ctx, -1), lambda: ops_amd.cache_read(kc, bt, ctx, 1 << 31),
        lambda: ops_amd.cache_read(k8, bt, ctx, 4), lambda: ops_amd.cache_read(kc, bt, ctx, 4, scales=s8),
        lambda: ops_amd.cache_read(kc.half(), bt, ctx, 4), lambda: ops_amd.cache_read(kc, bt, ctx, 4, dtype=torch.float16),
        lambda: ops_amd.cache_read(kc, bt, ctx[:1], 4), lambda: ops_amd.cache_read(kc, bt, ctx, 4, ctx[:1]),
        lambda: ops_amd.cache_read(kc, bt[0], ctx, 4), lambda: ops_amd.cache_read(kc[0], bt, ctx, 4),
        lambda: ops_amd.cache_read(kc, bt, ctx, 4, out=torch.zeros(2, 5, 2, 64)),
        lambda: ops_amd.cache_read(kc.clone().requires_grad_(True), bt, ctx, 4),
        lambda: ops_amd.cache_read(kc, bt, ctx, 4, out=torch.zeros(2, 4, 2, 1).expand(2, 4, 2, 64)),
    ]
    for c in calls:
        with pytest.raises(ValueError):
            c()
    assert launches == []
    wide = torch.zeros(1, 16, 1, 64).expand((1 << 32) + 1, 16, 1, 64)
    with pytest.raises(ValueError, match="past 2"):
        chunk(k=wide, v=wide)
    with pytest.raises(ValueError, match="past 2"):
        ops_amd.cache_read(wide, bt, ctx, 4)


def test_cpu_tensors_are_refused():
    q, kc, bt, i = torch.randn(1, 2, 4, 64), torch.randn(4, 16, 2, 64), torch.zeros(1, 1, dtype=I32), torch.zeros(1, dtype=I32)
    for c in (lambda: ops_amd.chunk_attention_paged(q, kc, kc, bt, i), lambda: ops_amd.window_attention(q, q, q),
              lambda: ops_amd.cache_read(kc, bt, i, 3)):
        with pytest.raises(ValueError, match="GPU"):
            c()


def test_what_autograd_is_told(launches):
    """The tensors that a call writes count as changed for graphs that have saved them."""
    kc, s8 = torch.zeros(9, 16, 2, 64).to(F8), torch.zeros(9, 16, 2, dtype=torch.uint8)
    x, bt, pos = torch.randn(2, 3, 2, 64), torch.zeros(2, 2, dtype=I32), torch.arange(3)
    v0 = kc._version, s8._version
    ops_amd.qk_norm_rope_append(None, x, None, kc, None, bt, pos, pos, ops_amd.rope_frequencies(64), k_scales=s8)
    assert kc._version > v0[0] and s8._version > v0[1]
    q = torch.randn(2, 3, 4, 64, requires_grad=True)
    k = torch.randn(2, 3, 2, 64)
    out, _ = ops_amd.window_attention(q, k, k)
    k.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
