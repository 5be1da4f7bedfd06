"""GPU tests of the drafted-tree attention against float64.

Tolerances: a score is a float32 sum of D products, off by at most (D + 8) 2^-24
max_s scale sum |q k| = d; a weight p is then off by 2 d relatively, and
rounding the weights to bfloat16 for the matrix cores adds finfo.eps / 2 = 2^-8
(float32: none).  So |out - ref| <= eps/2 |ref| + (2 d + w + 2^-20) sum p |v|, with w = 2^-8
or 0, and |lse - ref| <= d + 2^-21 (1 + |ref|)."""
import math
import random

import pytest
import torch

import ops_amd
from tests import ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def _g(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _masks(B, T, seed, empty=()):
    r = random.Random(seed)
    m = []
    for _ in range(B):
        row = [1]
        for i in range(1, T):
            x = row[max(0, i - r.randint(1, 4))] | (1 << i)
            row.append(x)
        m.append(row)
    for b, t in empty:
        m[b][t] = 0
    return torch.tensor([[x - (1 << 64) if x >= 1 << 63 else x for x in row] for row in m], dtype=torch.int64, device=DEV)


def _pool(g, B, maxp, ps, Hkv, Dk, Dv, dt, shared):
    n = B * maxp + 3
    kc = torch.randn(n, ps, Hkv, Dk, generator=g, device=DEV).to(dt)
    vc = kc[..., :Dv] if shared else torch.randn(n, ps, Hkv, Dv, generator=g, device=DEV).to(dt)
    bt = torch.randperm(n, generator=g, device=DEV)[:B * maxp].view(B, maxp).to(torch.int32)
    return kc, vc, bt


def _check(q, kc, vc, bt, ctx, mask, nodes, scale, sink, out, lse):
    o, l, pv, mag = ref.tree(q, kc, vc, bt, ctx, mask, nodes, scale, sink)
    D = q.shape[3]
    d = (D + 8) * 2.0 ** -24 * mag
    w = 2.0 ** -8 if q.dtype == BF16 else 0.0
    assert torch.equal(torch.isfinite(lse), torch.isfinite(l))
    fin = torch.isfinite(l)
    if fin.any():
        assert float(((lse.double() - l).abs() - (d + 2.0 ** -21 * (1 + l.abs())))[fin].max()) <= 0.0
    assert torch.equal(lse[~fin].double(), l[~fin])
    bound = torch.finfo(q.dtype).eps / 2 * o.abs() + (2 * d[..., None] + w + 2.0 ** -20) * pv
    err = (out.double() - o).abs() - bound
    assert torch.isfinite(out).all()
    assert float(err.max()) <= 0.0, (float(err.max()), float((out.double() - o).abs().max()))


CASES = [
    # name, dtype, T, Hq, Hkv, Dk, Dv, shared, page, ctx, sink
    ("one-token", BF16, 1, 1, 1, 128, 128, False, 64, [0, 1, 63], False),
    ("d128-g8", BF16, 8, 16, 2, 128, 128, False, 64, [64, 65, 1000], False),
    ("d128-g16-t7-sink", BF16, 7, 16, 1, 128, 128, False, 16, [31, 200, 511], True),
    ("d128-t64", BF16, 64, 8, 2, 128, 128, False, 64, [5, 700], False),
    ("d128-g1", BF16, 5, 3, 3, 128, 128, False, 32, [100, 33, 2], False),
    ("d128-g17", BF16, 3, 17, 1, 128, 128, False, 64, [130, 64], True),
    ("d128-g128", BF16, 2, 128, 1, 128, 128, False, 64, [300], False),
    ("d64-g4", BF16, 16, 8, 2, 64, 64, False, 64, [999, 0, 128], True),
    ("d64-shared-kv", BF16, 9, 32, 1, 64, 64, True, 8, [77, 256], False),
    ("mla-128", BF16, 3, 128, 1, 576, 512, True, 64, [300, 31], False),
    ("mla-16", BF16, 8, 16, 1, 576, 512, True, 64, [129, 1], True),
    ("mla-1", BF16, 1, 1, 1, 576, 512, True, 16, [40], False),
    ("odd-dims", BF16, 4, 6, 2, 77, 33, False, 4, [50, 3], True),
    ("d192-v128", BF16, 4, 4, 2, 192, 128, False, 64, [200], False),
    ("f32-d64", F32, 6, 8, 2, 64, 64, False, 64, [300, 17], True),
    ("f32-d128-t64", F32, 64, 4, 1, 128, 128, False, 64, [65], False),
    ("f32-odd", F32, 3, 3, 1, 50, 70, False, 1, [11, 0], False),
    ("bf16-d1024", BF16, 2, 2, 1, 1024, 1024, False, 16, [40], False),
]


@pytest.mark.parametrize("c", CASES, ids=[c[0] for c in CASES])
def test_tree_attention(c):
    _, dt, T, Hq, Hkv, Dk, Dv, shared, ps, ctx, with_sink = c
    g = _g(1)
    B = len(ctx)
    maxp = (max(ctx) + T + ps - 1) // ps + 1
    kc, vc, bt = _pool(g, B, maxp, ps, Hkv, Dk, Dv, dt, shared)
    q = (2 * torch.randn(B, T, Hq, Dk, generator=g, device=DEV)).to(dt)
    mask = _masks(B, T, 2)
    sink = torch.randn(Hq, generator=g, device=DEV) if with_sink else None
    cl = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    nodes = torch.tensor([max(1, T - b) for b in range(B)], dtype=torch.int32, device=DEV)
    for n in (None, nodes):
        out, lse = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, n, attn_sink=sink)
        torch.cuda.synchronize()
        _check(q, kc, vc, bt, ctx, mask, n, 1 / math.sqrt(Dk), sink, out, lse)


KINDS = [("bf16-d128", BF16, 4, 16, 2, 128, 128, False), ("bf16-d64", BF16, 4, 8, 2, 64, 64, False),
         ("mla", BF16, 3, 16, 1, 576, 512, True), ("mla-128", BF16, 2, 128, 1, 576, 512, True),
         ("f32", F32, 4, 4, 2, 64, 64, False), ("odd", BF16, 3, 4, 2, 40, 24, False)]


@pytest.mark.parametrize("k", KINDS, ids=[k[0] for k in KINDS])
@pytest.mark.parametrize("with_sink", [False, True])
def test_rows_that_see_nothing(k, with_sink):
    """No context and an empty mask; a sequence without nodes; unmapped pages in
    the middle, at the end and throughout; lengths past the table or negative."""
    _, dt, T, Hq, Hkv, Dk, Dv, shared = k
    g = _g(3)
    ps, maxp = 16, 20
    ctx = [0, 250, 0, 300, 100, 5000, -7]
    B = len(ctx)
    kc, vc, bt = _pool(g, B, maxp, ps, Hkv, Dk, Dv, dt, shared)
    bt[3, 4:9] = -1
    bt[3, 18] = kc.shape[0]
    bt[4] = -1
    q = (2 * torch.randn(B, T, Hq, Dk, generator=g, device=DEV)).to(dt)
    mask = _masks(B, T, 4, empty=[(0, 0), (2, 1)])
    nodes = torch.tensor([T, 0, T, T, T, T, T + 5], dtype=torch.int32, device=DEV)
    sink = torch.randn(Hq, generator=g, device=DEV) if with_sink else None
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, bt, torch.tensor(ctx, dtype=torch.int32, device=DEV), mask, nodes,
                                            sm_scale=0.1, attn_sink=sink)
    torch.cuda.synchronize()
    _check(q, kc, vc, bt, ctx, mask, nodes, 0.1, sink, out, lse)
    assert float(out[1].abs().max()) == 0.0 and bool((lse[1] == -math.inf).all())
    if with_sink:
        assert torch.equal(lse[0, 0], sink)


@pytest.mark.parametrize("k", KINDS, ids=[k[0] for k in KINDS])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_unseen_rows_may_hold_anything(k, bad):
    """NaN and infinities in cache rows that a token does not see: behind the last
    node, on pages of no sequence, and in drafted rows that only other tokens see."""
    _, dt, T, Hq, Hkv, Dk, Dv, shared = k
    g = _g(5)
    ps, maxp, ctx, B = 16, 12, [37, 120], 2
    kc, vc, bt = _pool(g, B, maxp, ps, Hkv, Dk, Dv, dt, shared)
    q = (2 * torch.randn(B, T, Hq, Dk, generator=g, device=DEV)).to(dt)
    mask = torch.ones(B, T, dtype=torch.int64, device=DEV)
    mask[:, 1] = 2  # node 1 sees itself only, the others node 0 only
    nodes = torch.tensor([T, T - 1], dtype=torch.int32, device=DEV)
    cl = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    want, wl = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, nodes)
    ok = torch.ones(kc.shape[:2], dtype=torch.bool, device=DEV)
    for b in range(B):
        for i in list(range(ctx[b])) + [ctx[b]]:
            ok[int(bt[b, i // ps]), i % ps] = False
    kc[ok] = bad
    if not shared:
        vc[ok] = bad
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, nodes)
    torch.cuda.synchronize()
    rows = [t for t in range(T) if t != 1]
    assert torch.isfinite(out[:, rows].float()).all()
    err = (out[:, rows].double() - want[:, rows].double()).abs()
    # the same products, perhaps added in another order or with unrounded weights
    lim = 2.0 ** -6 if dt == BF16 else 2.0 ** -18
    assert float((err - lim * (1 + want[:, rows].double().abs())).max()) <= 0.0
    assert torch.equal(torch.isfinite(lse[:, rows]), torch.isfinite(wl[:, rows]))


def test_strides_and_preallocated_results():
    """A query of [B, Hq, T, D] layout, interleaved k and v pages, a table wider
    than its view, int64 table, results into slices of larger tensors."""
    g = _g(6)
    B, T, Hq, Hkv, D, ps, maxp = 2, 5, 8, 2, 128, 16, 9
    kv = torch.randn(B * maxp, 2, ps, Hkv, D, generator=g, device=DEV).to(BF16)
    kc, vc = kv[:, 0], kv[:, 1]
    bt = torch.randperm(B * maxp, generator=g, device=DEV).view(B, maxp)[:, :8]
    q = torch.randn(B, Hq, T, D, generator=g, device=DEV).to(BF16).transpose(1, 2)
    mask = _masks(B, T, 7).t().contiguous().t()
    ctx = [100, 77]
    cl = torch.tensor(ctx, device=DEV)
    big, bl = torch.zeros(B, T, 2 * Hq, D, dtype=BF16, device=DEV), torch.zeros(B, 2 * Hq, T, device=DEV)
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, out=big[:, :, Hq:], lse=bl[:, Hq:].transpose(1, 2))
    torch.cuda.synchronize()
    _check(q, kc, vc, bt, ctx, mask, None, 1 / math.sqrt(D), None, out, lse)
    assert float(big[:, :, :Hq].abs().max()) == 0.0 and float(bl[:, :Hq].abs().max()) == 0.0
    # a view with an odd offset: rows that are not 16-byte aligned
    odd = torch.randn(B * maxp, ps, Hkv, D + 1, generator=g, device=DEV).to(BF16)
    ko, vo = odd[..., 1:], odd[..., :D]
    out, lse = ops_amd.tree_attention_paged(q, ko, vo, bt, cl, mask)
    torch.cuda.synchronize()
    _check(q, ko, vo, bt, ctx, mask, None, 1 / math.sqrt(D), None, out, lse)


@pytest.mark.parametrize("Dk,Dv,Hq,Hkv", [(128, 128, 4, 2), (576, 512, 16, 1)])
def test_rows_far_into_a_large_pool(Dk, Dv, Hq, Hkv):
    """Pages past 2^31 elements (4 GiB) of the pool."""
    ps, T = 64, 3
    n = (1 << 31) // (ps * Hkv * Dk) + 6
    g = _g(8)
    kc = torch.empty(n, ps, Hkv, Dk, dtype=BF16, device=DEV)
    vc = kc[..., :Dv] if Dv < Dk else torch.empty(n, ps, Hkv, Dv, dtype=BF16, device=DEV)
    bt = torch.tensor([[n - 1, 0, n - 2, 1, n - 3]], dtype=torch.int32, device=DEV)
    for p in bt[0].tolist():
        kc[p] = torch.randn(ps, Hkv, Dk, generator=g, device=DEV).to(BF16)
        if Dv == Dk:
            vc[p] = torch.randn(ps, Hkv, Dv, generator=g, device=DEV).to(BF16)
    q = torch.randn(1, T, Hq, Dk, generator=g, device=DEV).to(BF16)
    ctx, mask = [300], _masks(1, T, 9)
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, bt, torch.tensor(ctx, device=DEV), mask)
    torch.cuda.synchronize()
    _check(q, kc, vc, bt, ctx, mask, None, 1 / math.sqrt(Dk), None, out, lse)


@pytest.mark.parametrize("k", KINDS, ids=[k[0] for k in KINDS])
def test_long_context_on_a_wide_table(k):
    """Many key ranges, ragged, on a table far wider than the contexts; twice bitwise the same."""
    _, dt, T, Hq, Hkv, Dk, Dv, shared = k
    g = _g(10)
    ps, ctx = 64, [9000, 1, 777, 4096]
    maxp = 256
    B = len(ctx)
    n = sum((c + T + ps - 1) // ps for c in ctx)
    kc = torch.randn(n, ps, Hkv, Dk, generator=g, device=DEV).to(dt)
    vc = kc[..., :Dv] if shared else torch.randn(n, ps, Hkv, Dv, generator=g, device=DEV).to(dt)
    bt = torch.full((B, maxp), -1, dtype=torch.int32, device=DEV)
    perm, at = torch.randperm(n, generator=g, device=DEV).to(torch.int32), 0
    for b, c in enumerate(ctx):
        m = (c + T + ps - 1) // ps
        bt[b, :m] = perm[at:at + m]
        at += m
    q = torch.randn(B, T, Hq, Dk, generator=g, device=DEV).to(dt)
    mask, cl = _masks(B, T, 11), torch.tensor(ctx, dtype=torch.int32, device=DEV)
    sink = torch.randn(Hq, generator=g, device=DEV)
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, attn_sink=sink)
    out2, lse2 = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, attn_sink=sink)
    torch.cuda.synchronize()
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    _check(q, kc, vc, bt, ctx, mask, None, 1 / math.sqrt(Dk), sink, out, lse)


def test_many_sequences():
    """More than 64 sequences: the key ranges are found over several steps."""
    g = _g(12)
    B, T, Hq, Hkv, D, ps = 150, 2, 4, 1, 64, 16
    ctx = [(37 * b) % 300 for b in range(B)]
    kc, vc, bt = _pool(g, B, 20, ps, Hkv, D, D, BF16, False)
    q = torch.randn(B, T, Hq, D, generator=g, device=DEV).to(BF16)
    mask, cl = _masks(B, T, 13), torch.tensor(ctx, dtype=torch.int32, device=DEV)
    out, lse = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask)
    torch.cuda.synchronize()
    _check(q, kc, vc, bt, ctx, mask, None, 1 / math.sqrt(D), None, out, lse)


def test_captured_calls_follow_their_inputs():
    """Two captured calls, replayed in turn with eager work between; lengths and
    tables change on the device between replays."""
    g = _g(14)
    B, T, Hq, Hkv, D, ps, maxp = 3, 4, 16, 2, 128, 64, 40
    kc, vc, bt = _pool(g, B, maxp, ps, Hkv, D, D, BF16, False)
    q = torch.randn(B, T, Hq, D, generator=g, device=DEV).to(BF16)
    mask, cl = _masks(B, T, 15), torch.tensor([100, 900, 5], dtype=torch.int32, device=DEV)

    def f():
        return ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(f())
        graphs.append(gr)
    for ctx in ([100, 900, 5], [2000, 0, 64], [1, 2, 2500]):
        cl.copy_(torch.tensor(ctx, dtype=torch.int32))
        want = f()
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
