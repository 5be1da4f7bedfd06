"""GPU tests of the drafted-tree attention's forms for pages that hold whole tiles
and for row counts of every kernel, against float64 (tolerances as derived in
test_gpu_tree.py): NaN and infinities in rows that a token does not see, joins
of many slots, one range a sequence, results that autograd has to know of."""
import math

import pytest
import torch

import ops_amd
from tests import ops_ref as ref
from tests.test_gpu_tree import BF16, CASES, DEV, F32, _check, _g, _masks, _pool

pytestmark = pytest.mark.gpu

# name, dtype, T, Hq, Hkv, Dk, Dv, shared: rows T Hq / Hkv of each kernel
KINDS = [("rows16", BF16, 4, 8, 2, 128, 128, False), ("rows32", BF16, 4, 8, 1, 64, 64, False),
         ("rows64", BF16, 8, 16, 2, 128, 128, False), ("rows128", BF16, 8, 16, 1, 128, 128, False),
         ("rows128-d64", BF16, 20, 12, 2, 64, 64, False), ("rows256", BF16, 30, 14, 2, 128, 128, False),
         ("rows512-d64", BF16, 64, 8, 1, 64, 64, False), ("mla-64", BF16, 4, 16, 1, 576, 512, True),
         ("mla-200", BF16, 5, 40, 1, 576, 512, True), ("f32", F32, 4, 4, 2, 64, 64, False)]


def _wide(bt, ps):
    """The table with room for 2^17 rows: the kernels of many rows a workgroup,
    which short tables leave to those of 16 and 32."""
    return torch.cat((bt, torch.full((bt.shape[0], (1 << 17) // ps), -1, dtype=torch.int32, device=DEV)), 1)


@pytest.mark.parametrize("c", CASES, ids=[c[0] for c in CASES])
def test_wide_tables(c):
    _, dt, T, Hq, Hkv, Dk, Dv, shared, ps, ctx, with_sink = c
    g = _g(27)
    B = len(ctx)
    kc, vc, bt = _pool(g, B, (max(ctx) + T + ps - 1) // ps + 1, ps, Hkv, Dk, Dv, dt, shared)
    q = (2 * torch.randn(B, T, Hq, Dk, generator=g, device=DEV)).to(dt)
    mask, cl = _masks(B, T, 28), torch.tensor(ctx, dtype=torch.int32, device=DEV)
    sink = torch.randn(Hq, generator=g, device=DEV) if with_sink else None
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, _wide(bt, ps), cl, mask, attn_sink=sink)
    torch.cuda.synchronize()
    _check(q, kc, vc, bt, ctx, mask, None, 1 / math.sqrt(Dk), sink, out, lse)


@pytest.mark.parametrize("k", KINDS, ids=[k[0] for k in KINDS])
@pytest.mark.parametrize("ps", [16, 32, 64, 256])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("bad", [math.nan, -math.inf])
def test_unseen_rows_of_a_page_may_hold_anything(k, ps, wide, bad):
    _, dt, T, Hq, Hkv, Dk, Dv, shared = k
    g = _g(21)
    ctx = [37, 192, 700]
    B = len(ctx)
    maxp = (max(ctx) + T + ps - 1) // ps + 1
    kc, vc, bt = _pool(g, B, maxp, ps, Hkv, Dk, Dv, dt, shared)
    q = (2 * torch.randn(B, T, Hq, Dk, generator=g, device=DEV)).to(dt)
    mask = torch.ones(B, T, dtype=torch.int64, device=DEV)
    mask[:, 1] = 2  # node 1 sees itself only, the others node 0 only
    nodes = torch.tensor([T, T - 1, T], dtype=torch.int32, device=DEV)
    cl = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    scale = 1 / math.sqrt(Dk)
    o, l, pv, mag = ref.tree(q, kc, vc, bt, ctx, mask, nodes, scale, None)  # (of the clean cache)
    ok = torch.ones(kc.shape[:2], dtype=torch.bool, device=DEV)
    for b in range(B):
        for i in range(ctx[b] + 1):
            ok[int(bt[b, i // ps]), i % ps] = False
    kc[ok] = bad
    if not shared:
        vc[ok] = bad
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, _wide(bt, ps) if wide else bt, cl, mask, nodes)
    torch.cuda.synchronize()
    rows = [t for t in range(T) if t != 1]
    out, lse, o, l, pv, mag = (x[:, rows].double() for x in (out, lse, o, l, pv, mag))
    assert torch.isfinite(out).all()
    assert torch.equal(torch.isfinite(lse), torch.isfinite(l))
    fin = torch.isfinite(l)
    d = (Dk + 8) * 2.0 ** -24 * mag
    w = 2.0 ** -8 if dt == BF16 else 0.0
    assert float(((lse - l).abs() - (d + 2.0 ** -21 * (1 + l.abs())))[fin].max()) <= 0.0
    bound = torch.finfo(dt).eps / 2 * o.abs() + (2 * d[..., None] + w + 2.0 ** -20) * pv
    assert float(((out - o).abs() - bound).max()) <= 0.0


@pytest.mark.parametrize("dt,T,Hq,Hkv,Dk,Dv,shared", [
    (BF16, 1, 2, 1, 128, 128, False), (BF16, 3, 4, 1, 64, 64, False), (F32, 1, 2, 1, 50, 70, False),
    (BF16, 1, 3, 1, 192, 300, False), (BF16, 1, 16, 1, 576, 512, True), (F32, 2, 1, 1, 20, 516, False)])
@pytest.mark.parametrize("with_sink", [False, True])
def test_many_slots_of_few_rows(dt, T, Hq, Hkv, Dk, Dv, shared, with_sink):
    g = _g(22)
    ps, ctx = 64, [30011, 3]
    kc, vc, bt = _pool(g, 2, 480, ps, Hkv, Dk, Dv, dt, shared)
    q = (2 * torch.randn(2, T, Hq, Dk, generator=g, device=DEV)).to(dt)
    mask, cl = _masks(2, T, 23), torch.tensor(ctx, dtype=torch.int32, device=DEV)
    sink = torch.randn(Hq, generator=g, device=DEV) if with_sink else None
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, attn_sink=sink)
    torch.cuda.synchronize()
    _check(q, kc, vc, bt, ctx, mask, None, 1 / math.sqrt(Dk), sink, out, lse)


def test_one_range_a_sequence():
    """More sequences than ranges in flight; some without keys or nodes."""
    g = _g(24)
    B, T, Hq, Hkv, D, ps = 300, 1, 4, 2, 64, 32
    ctx = [(53 * b) % 200 if b % 7 else 0 for b in range(B)]
    kc, vc, bt = _pool(g, B, 8, ps, Hkv, D, D, BF16, False)
    q = torch.randn(B, T, Hq, D, generator=g, device=DEV).to(BF16)
    nodes = torch.tensor([b % 3 != 0 for b in range(B)], dtype=torch.int32, device=DEV)
    mask, cl = _masks(B, T, 25), torch.tensor(ctx, dtype=torch.int32, device=DEV)
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, nodes)
    torch.cuda.synchronize()
    _check(q, kc, vc, bt, ctx, mask, nodes, 1 / math.sqrt(D), None, out, lse)


def test_tensors_that_are_written():
    g = _g(26)
    x = torch.randn(1, 4, 2, 64, generator=g, device=DEV)
    pos, freq = torch.arange(4, device=DEV), ops_amd.rope_frequencies(64, device=DEV)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = (x * w).sum()  # saves x
    ops_amd.rotary_embedding(x, pos, freq, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with pytest.raises(ValueError, match="expanded"):
        ops_amd.rotary_embedding(x, pos, freq, out=x[:, :, :1].expand(1, 4, 2, 64))
    kc, vc, bt = _pool(g, 1, 4, 16, 1, 64, 64, F32, False)
    cl, mask = torch.tensor([20], dtype=torch.int32, device=DEV), torch.ones(1, 4, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="expanded"):
        ops_amd.tree_attention_paged(x, kc, vc, bt, cl, mask, lse=torch.empty(1, 4, 1, device=DEV).expand(1, 4, 2))
    with pytest.raises(ValueError, match="twice"):
        ops_amd.cache_keep_path([kc, kc], bt, cl, torch.zeros(1, 2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="expanded"):
        ops_amd.cache_free(bt.expand(2, -1) if bt.shape[0] == 1 else bt[:1].expand(2, -1),
                           torch.ones(7, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="gradient"):
        ops_amd.cache_copy_pages([kc.clone().requires_grad_(True)], bt[0, :1], bt[0, 1:2])
