"""Dense attention of a chunk over a paged cache: kernels against float64
(tests/dense_ref.py derives the tolerances)."""
import math

import pytest
import torch

import ops_amd
from tests import dense_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _case(dtype=BF, fp8=False, S=5, ctx=(40, 0, 130), n=None, Hq=8, Hkv=2, D=64, Dv=None, page=16, seed=0, mla=False, extra=0):
    """q, caches, scales, table, ctx, lens; the pool's rows that no sequence holds are NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, Dv = len(ctx), D if Dv is None else Dv
    lens = [c + S for c in ctx]
    num = sum((x + page - 1) // page for x in lens) + 3
    bt = ref.table(lens, page, num, seed, extra)
    q = 2.0 * torch.randn(B, S, Hq, D, generator=g, device=DEV).to(dtype)
    k = torch.randn(num, page, Hkv, D, generator=g, device=DEV).to(dtype)
    v = k[..., :Dv] if mla else torch.randn(num, page, Hkv, Dv, generator=g, device=DEV).to(dtype)
    held = torch.zeros(num * page, dtype=torch.bool, device=DEV)
    at = torch.arange(bt.shape[1] * page, device=DEV)
    for b, x in enumerate(lens):
        m = x if n is None else ctx[b] + min(max(n[b], 0), S)
        held[(bt[b, at[:m] // page].long() * page + at[:m] % page)] = True
    ks = vs = None
    if fp8:
        k, ks = ref.quantised(k)
        v, vs = (k[..., :Dv], ks) if mla else ref.quantised(v)
    (k.view(torch.uint8) if fp8 else k).view(num * page, -1)[~held] = 0x7f if fp8 else math.nan
    if not mla:
        (v.view(torch.uint8) if fp8 else v).view(num * page, -1)[~held] = 0x7f if fp8 else math.nan
    ctx = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    n = None if n is None else torch.tensor(n, dtype=torch.int32, device=DEV)
    return dict(q=q, k=k, v=v, ks=ks, vs=vs, bt=bt, ctx=ctx, n=n)


def _run(c, **kw):
    return ops_amd.chunk_attention_paged(c["q"], c["k"], c["v"], c["bt"], c["ctx"], c["n"], k_scales=c["ks"], v_scales=c["vs"], **kw)


def _want(c, window=None, first=0, attn_sink=None, sm_scale=None):
    return ref.chunk(c["q"], c["k"], c["v"], c["bt"], c["ctx"], c["n"], window, first, attn_sink, c["ks"], c["vs"], sm_scale)


def _w(c):
    """Weights are rounded to bf16 where the matrix cores take bf16 products."""
    return 2.0 ** -8 if c["q"].dtype == BF else 0.0


def _both(c, **kw):
    got = _run(c, **kw)
    ref.check(got, _want(c, **kw), c["q"].shape[3], c["q"].dtype, _w(c))
    return got


FORMS = [("bf16", BF, False), ("f32", F32, False), ("bf16-e4m3", BF, True), ("f32-e4m3", F32, True)]
forms = pytest.mark.parametrize("dtype,fp8", [f[1:] for f in FORMS], ids=[f[0] for f in FORMS])


@forms
@pytest.mark.parametrize("D,Dv", [(64, 64), (128, 128), (96, 40), (20, 12), (33, 7), (192, 128), (256, 256)])
def test_head_dims(dtype, fp8, D, Dv):
    _both(_case(dtype, fp8, D=D, Dv=Dv))


@forms
def test_latent_rows(dtype, fp8):
    c = _case(dtype, fp8, D=576, Dv=512, Hq=16, Hkv=1, mla=True, S=7, ctx=(70, 3))
    got = _both(c)
    if fp8:  # v_scales may be left out
        c["vs"] = None
        again = _run(c)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@forms
@pytest.mark.parametrize("S", [1, 2, 31, 65, 200])
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (16, 2), (40, 2)])
def test_chunks_and_heads(dtype, fp8, S, heads):
    _both(_case(dtype, fp8, S=S, ctx=(0, 100), Hq=heads[0], Hkv=heads[1], D=64 if S > 2 else 128, seed=S))


@forms
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 3), (16, 0), (33, 4), (64, 64), (100, 1), (1000, 4), (7, 1000), (None, 5),
                                          ((1 << 31) - 1, (1 << 31) - 1)])
def test_windows(dtype, fp8, D, window, first):
    _both(_case(dtype, fp8, S=70, ctx=(300, 0, 31), D=D, Hq=4, Hkv=2), window=window, first=first)


@forms
def test_padding_and_empty_rows(dtype, fp8):
    """Sequences without tokens, tokens past a sequence's, sequences without a page."""
    c = _case(dtype, fp8, S=9, ctx=(40, 0, 130, 20), n=[9, 0, 4, -3])
    sink = torch.randn(8, device=DEV)
    for kw in (dict(), dict(attn_sink=sink), dict(window=5, first=2, attn_sink=sink)):
        out, lse = _both(c, **kw)
        for b, n in enumerate((9, 0, 4, 0)):
            assert float(out[b, n:].abs().sum()) == 0.0 and bool((lse[b, n:] == -math.inf).all())
    c["bt"] = torch.full_like(c["bt"], -1)
    out, lse = _both(c)
    assert float(out.abs().sum()) == 0.0 and bool((lse == -math.inf).all())
    out, lse = _both(c, attn_sink=sink)
    assert torch.equal(lse[0], sink.expand(9, 8))


@forms
@pytest.mark.parametrize("page", [1, 2, 8, 32, 64, 256])
def test_pages(dtype, fp8, page):
    """Page sizes, pages that are not mapped or outside of the pool, int64 tables and lengths."""
    c = _case(dtype, fp8, S=12, ctx=(100, 0, 77), page=page, extra=2)
    for e, x in ((3, -1), (1, 10 ** 6), (0, -7)):
        c["bt"][0, min(e, c["bt"].shape[1] - 1)] = x
    got = _both(c, window=50, first=20)
    c["bt"], c["ctx"] = c["bt"].long(), c["ctx"].long()
    again = _run(c, window=50, first=20)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@forms
def test_context_past_the_table(dtype, fp8):
    """Lengths past the table and below 0 are those of its end and start."""
    c = _case(dtype, fp8, S=6, ctx=(58, 20), n=[6, 6], page=16)
    c["ctx"] = torch.tensor([10 ** 6, -5], dtype=torch.int32, device=DEV)
    (c["k"].view(torch.uint8) if fp8 else c["k"]).zero_()
    (c["v"].view(torch.uint8) if fp8 else c["v"]).zero_()
    _both(c)


@pytest.mark.parametrize("dtype,fp8", [(BF, False), (F32, False), (BF, True)])
@pytest.mark.parametrize("D", [64, 128, 576])
def test_masked_infinities(dtype, fp8, D):
    """Rows that a token does not see may hold anything: later tokens, rows left of the
    window; the tokens that do see them get what the formula gives."""
    S, ctx = 40, 90
    c = _case(dtype, fp8, S=S, ctx=(ctx,), n=[S], Hq=4, Hkv=1, D=D, Dv=512 if D == 576 else D, mla=D == 576, page=32)
    plain = _both(c, window=50, first=4)
    for j in (10, ctx + 20):  # left of every window; seen from token 20 on
        p, r = int(c["bt"][0, j // 32]), j % 32
        for t in (c["k"], c["v"]):
            if fp8:
                t.view(torch.uint8)[p, r] = 0x7f
            else:
                t[p, r] = math.inf
                t[p, r, :, 1::2] = math.nan
    out, lse = _run(c, window=50, first=4)
    assert torch.equal(out[0, :20], plain[0][0, :20]) and torch.equal(lse[0, :20], plain[1][0, :20])
    assert bool(torch.isnan(out[0, 20:]).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_infinite_values_that_are_seen(dtype):
    """An infinite v element reaches its dim of the tokens that see it and no other."""
    S, ctx = 20, 50
    c = _case(dtype, S=S, ctx=(ctx,), Hq=4, Hkv=1, D=64, page=32)
    plain = _run(c)[0]
    p, r = int(c["bt"][0, (ctx + 7) // 32]), (ctx + 7) % 32
    c["v"][p, r, 0, 5] = math.inf
    out = _run(c)[0]
    assert bool((out[0, 7:, :, 5] == math.inf).all()) and torch.equal(out[0, :7], plain[0, :7])
    out[0, 7:, :, 5] = plain[0, 7:, :, 5]
    assert torch.equal(out, plain)


@forms
@pytest.mark.parametrize("D", [64, 128])
def test_many_ranges(dtype, fp8, D):
    """Few rows over long contexts: the keys are cut into ranges and joined."""
    c = _case(dtype, fp8, S=1, ctx=(9000, 17, 0, 4100), Hq=8, Hkv=2, D=D, page=64)
    sink = torch.randn(8, device=DEV)
    _both(c)
    _both(c, window=3000, first=130, attn_sink=sink)
    _both(_case(dtype, fp8, S=33, ctx=(5000, 1), n=[33, 20], Hq=4, Hkv=1, D=D, page=64))


@forms
def test_strides(dtype, fp8):
    """Views of wider tensors, permuted outputs, odd offsets, q without a unit stride."""
    for off in (0, 1, 8):
        c = _case(dtype, fp8, S=6, ctx=(40, 9), D=64)
        want = _run(c)
        wide = torch.zeros(*c["q"].shape[:3], 64 + 16, dtype=dtype, device=DEV)
        q = wide[..., off:off + 64]
        q.copy_(c["q"])
        pool = torch.zeros(*c["k"].shape[:2], 64 + 16, 4, dtype=torch.uint8 if fp8 else dtype, device=DEV).transpose(2, 3).contiguous()
        k = pool[:, :, 1:3, off:off + 64]
        k.copy_(c["k"].view(torch.uint8) if fp8 else c["k"])
        k = k.view(F8) if fp8 else k
        out = torch.empty(6, 2, 8, 64 + 16, dtype=dtype, device=DEV).transpose(0, 1)[..., off:off + 64]
        lse = torch.empty(8, 6, 2, device=DEV).permute(2, 1, 0)
        d = dict(c, q=q, k=k)
        if fp8:
            d["ks"] = torch.stack((c["ks"], c["ks"]), -1)[..., 0]
        _run(d, out=out, lse=lse)
        ref.check((out, lse), _want(c), 64, dtype, _w(c))
        q2 = c["q"].transpose(2, 3).contiguous().transpose(2, 3)
        again = _run(dict(c, q=q2))
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_equal_calls_give_equal_bits():
    for S, ctx in ((1, (9000, 50)), (300, (1000, 0))):
        c = _case(S=S, ctx=ctx, D=128, page=64)
        a, b = _run(c), _run(c)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_other_scales():
    c = _case(S=17, D=128)
    for s in (1e-3, 0.5):
        _both(c, sm_scale=s)


def test_empty_batches():
    c = _case(S=3, ctx=(10,))
    out, lse = ops_amd.chunk_attention_paged(c["q"][:, :0], c["k"], c["v"], c["bt"], c["ctx"])
    assert out.shape == (1, 0, 8, 64) and lse.shape == (1, 0, 8)
    out, lse = ops_amd.chunk_attention_paged(c["q"][:0], c["k"], c["v"], c["bt"][:0], c["ctx"][:0])
    assert out.shape == (0, 3, 8, 64)
