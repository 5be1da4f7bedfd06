"""GPU tests of how many bits the drafted-tree attention's weights keep, kernel by
kernel: up to 64 rows a workgroup (d = 64 and 128) they are multiplied as two
bfloat16 parts, off by 2^-8 of 2^-8 = 2^-16 at most, and the kernel of other sizes
keeps them in float32.  One bfloat16 part is further off than the tolerance here,
which the tests show on the same inputs."""
import math

import pytest
import torch

import ops_amd
from tests.test_gpu_tree import BF16, DEV, F32, _g, _masks, _pool
from tests.test_gpu_tree_pages import _wide
from tests.tree_exact import bound, check, exact

pytestmark = pytest.mark.gpu

CASES = [  # name, dtype, T, Hq, Hkv, Dk, Dv, page, ctx, wide table
    ("rows16-d128", BF16, 8, 4, 2, 128, 128, 64, [300, 77], False), ("rows16-d64", BF16, 1, 4, 1, 64, 64, 16, [511, 3], False),
    ("rows16-of-many", BF16, 16, 16, 1, 128, 128, 64, [600], False),
    ("rows32-d128", BF16, 16, 4, 2, 128, 128, 16, [257, 640], True), ("rows32-d64", BF16, 8, 8, 2, 64, 64, 64, [480, 9], True),
    ("rows64-d128", BF16, 8, 16, 2, 128, 128, 64, [333, 900, 64], True),
    ("rows64-d64", BF16, 16, 16, 4, 64, 64, 32, [450, 31], True),
    ("other-dims", BF16, 4, 6, 2, 96, 80, 16, [300, 40], False), ("latent-of-a-copy", BF16, 2, 8, 1, 576, 512, 64, [130], False),
    ("f32-d64", F32, 4, 8, 2, 64, 64, 64, [300, 17], False)]


def _rounded(p):
    return p.float().to(BF16).double()


def _one_part_would_be_seen(args, want, D, dtype, w, n):
    """With weights rounded once, some results would be past the tolerance: the
    mistake is planted in the float64 values, on the CPU."""
    args = [x.cpu() if isinstance(x, torch.Tensor) else x for x in args]
    o, _, pv, mag = (x.cpu() for x in want)
    once = exact(*args, weights=_rounded)[0].to(dtype).double()
    return bool(((once - o).abs() > bound(o, pv, (D + 8) * 2.0 ** -24 * mag, dtype, w, n)).any())


@pytest.mark.parametrize("c", CASES, ids=[c[0] for c in CASES])
def test_weights_keep_their_bits(c):
    _, dt, T, Hq, Hkv, Dk, Dv, ps, ctx, wide = c
    g = _g(61)
    kc, vc, bt = _pool(g, len(ctx), (max(ctx) + T + ps - 1) // ps + 1, ps, Hkv, Dk, Dv, dt, False)
    q = torch.randn(len(ctx), T, Hq, Dk, generator=g, device=DEV).to(dt)
    mask, cl, scale = _masks(len(ctx), T, 62), torch.tensor(ctx, dtype=torch.int32, device=DEV), 1 / math.sqrt(Dk)
    got = ops_amd.tree_attention_paged(q, kc, vc, _wide(bt, ps) if wide else bt, cl, mask)
    torch.cuda.synchronize()
    w = 2.0 ** -16 if dt == BF16 and Dk == Dv and Dk in (64, 128) else 0.0
    args = (q, kc, vc, bt, ctx, mask, None, scale)
    want = exact(*args)
    check(got, want, Dk, dt, w, max(ctx))
    # (at 576 dims the scores' own bound, 2 (576 + 8) 2^-24 of 17 = 2^-9.7, is as large as one
    # part's rounding: there the value is checked, and one part would pass)
    assert Dk > 128 or _one_part_would_be_seen(args, want, Dk, dt, w, max(ctx))


@pytest.mark.parametrize("T,Hq,Hkv,D,wide", [(8, 2, 1, 128, False), (16, 2, 1, 64, True), (8, 16, 2, 128, True), (32, 4, 2, 64, True)])
def test_a_maximum_that_moves_inside_a_tile(T, Hq, Hkv, D, wide):
    """Scores climb by 9 (base 2) at key 20 of the first tile of 32, at key 50, 85 and so on:
    the running maximum moves between the two halves of a tile, after the first
    half's weights are held in two parts, and both parts have to follow."""
    g = _g(63)
    ps, ctx = 64, [300, 205]
    kc, vc, bt = _pool(g, 2, 6, ps, Hkv, D, D, BF16, False)
    kc *= 0.1
    u = torch.ones(D, device=DEV)
    q = (u + 0.1 * torch.randn(2, T, Hq, D, generator=g, device=DEV)).to(BF16)
    scale = 1 / math.sqrt(D)
    step = 9 * math.log(2) / (scale * D)  # of u: 9 in base-2 scores
    for b, c in enumerate(ctx):
        level = 0
        for s in range(c):
            level += s in (20, 50, 85, 127, 148, 210, 247)
            kc[int(bt[b, s // ps]), s % ps] = (kc[int(bt[b, s // ps]), s % ps].float() + step * level * (s % 16 in (4, 5, 2))).to(BF16)
    mask, cl = _masks(2, T, 64), torch.tensor(ctx, dtype=torch.int32, device=DEV)
    got = ops_amd.tree_attention_paged(q, kc, vc, _wide(bt, ps) if wide else bt, cl, mask)
    torch.cuda.synchronize()
    check(got, exact(q, kc, vc, bt, ctx, mask, None, scale), D, BF16, 2.0 ** -16, max(ctx))
