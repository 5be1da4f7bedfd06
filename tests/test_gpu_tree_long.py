"""GPU tests of the drafted-tree attention on key ranges of many tiles, against
float64: the kernels of 128 and 256 rows a workgroup and the one of latent rows
keep 2 to 5 tiles in flight, and a range has many times as many here, so every
stage of their rings is loaded, read and loaded again.  Pages in and outside of the
pool's range in the middle of a range, contexts that end inside a tile."""
import math

import pytest
import torch

import ops_amd
from tests.test_gpu_tree import BF16, DEV, _g, _masks
from tests.tree_exact import check, exact, slots

pytestmark = pytest.mark.gpu

STAGES = 5  # of the deepest ring; a step of these kernels takes 32 or 64 keys

KINDS = [  # name, T, Hq, Hkv, Dk, Dv, shared
    ("rows128-d128", 8, 128, 8, 128, 128, False), ("rows128-d64", 7, 96, 6, 64, 64, False),
    ("rows256-d128", 32, 64, 8, 128, 128, False), ("rows256-d64", 12, 128, 8, 64, 64, False),
    ("rows512-d128", 64, 32, 4, 128, 128, False), ("mla-512", 8, 64, 1, 576, 512, True),
    ("mla-130", 2, 65, 1, 576, 512, True)]
CTX = {"ragged": [8195, 20001, 12288, 9999], "even": [12224, 12256, 12288, 12320, 12352]}


def _batch(g, ctx, T, Hq, Hkv, Dk, Dv, shared, ps, wide=0):
    B = len(ctx)
    need = [(c + T + ps - 1) // ps for c in ctx]
    n = sum(need) + 2
    kc = torch.randn(n, ps, Hkv, Dk, generator=g, device=DEV).to(BF16)
    vc = kc[..., :Dv] if shared else torch.randn(n, ps, Hkv, Dv, generator=g, device=DEV).to(BF16)
    bt = torch.full((B, max(need) + wide), -1, dtype=torch.int32, device=DEV)
    perm, at = torch.randperm(n, generator=g, device=DEV).to(torch.int32), 0
    for b, m in enumerate(need):
        bt[b, :m] = perm[at:at + m]
        at += m
    q = (2 * torch.randn(B, T, Hq, Dk, generator=g, device=DEV)).to(BF16)
    return q, kc, vc, bt, torch.tensor(ctx, dtype=torch.int32, device=DEV)


def _run(q, kc, vc, bt, cl, ctx, mask, nodes, sink, longest):
    scale = 1 / math.sqrt(q.shape[3])
    got = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, nodes, attn_sink=sink)
    again = ops_amd.tree_attention_paged(q, kc, vc, bt, cl, mask, nodes, attn_sink=sink)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    check(got, exact(q, kc, vc, bt, ctx, mask, nodes, scale, sink), q.shape[3], BF16, 2.0 ** -8, longest)


@pytest.mark.parametrize("k", KINDS, ids=[k[0] for k in KINDS])
@pytest.mark.parametrize("ps", [16, 64, 256])
@pytest.mark.parametrize("lens", sorted(CTX))
def test_ranges_of_many_tiles(k, ps, lens):
    _, T, Hq, Hkv, Dk, Dv, shared = k
    g, ctx = _g(51), CTX[lens]
    q, kc, vc, bt, cl = _batch(g, ctx, T, Hq, Hkv, Dk, Dv, shared, ps, wide=3)
    # the average range (the longest is no shorter) in steps of 64 keys
    assert sum(ctx) / slots(q, kc, vc, bt) / 64 >= (2 * STAGES if Hkv > 1 or T > 2 else 3)
    for b in range(len(ctx)):  # unmapped, outside of the pool
        bt[b, (4000 + 700 * b) // ps] = -1
        bt[b, (7000 - 300 * b) // ps] = kc.shape[0]
    nodes = torch.tensor([T - b % 2 for b in range(len(ctx))], dtype=torch.int32, device=DEV)
    sink = torch.randn(Hq, generator=g, device=DEV) if lens == "even" else None
    _run(q, kc, vc, bt, cl, ctx, _masks(len(ctx), T, 52), nodes, sink, max(ctx))


@pytest.mark.parametrize("T,Hq,Hkv,D", [(8, 128, 8, 64), (16, 128, 8, 64)], ids=["rows128", "rows256"])
def test_one_range_a_sequence_of_many_tiles(T, Hq, Hkv, D):
    """More sequences than ranges wanted: each is one range, ended by its own length."""
    g = _g(53)
    ctx = [1500 + 37 * b for b in range(40)]
    q, kc, vc, bt, cl = _batch(g, ctx, T, Hq, Hkv, D, D, False, 64)
    assert slots(q, kc, vc, bt) == len(ctx) and min(ctx) / 64 >= 2 * STAGES
    bt[::3, 9] = -1
    _run(q, kc, vc, bt, cl, ctx, _masks(len(ctx), T, 54), None, None, max(ctx))
