"""How many bits the weights of dense attention keep, kernel by kernel: up to 64 rows a
workgroup (64 and 128 dims) they are multiplied as two bfloat16 parts, off by 2^-8 of 2^-8 =
2^-16 at most; other head dims keep them in float32, in the backward too.  One bfloat16 part
is further off than the tolerances here, which the tests show on the same inputs."""
import math

import pytest
import torch

import ops_amd
from tests import dense_ref as ref
from tests.test_gpu_dense import BF, DEV, F32, _case, _run, _want
from tests.test_gpu_window import _leaves
from tests.test_gpu_window import _run as _run_window

pytestmark = pytest.mark.gpu

CASES = [  # name, e4m3, S, heads, kv heads, D, Dv, page, ctx, bits of a weight
    ("rows16-d128", False, 1, 8, 2, 128, 128, 64, (300, 77), 16), ("rows16-d64", False, 2, 8, 2, 64, 64, 16, (511, 30), 16),
    ("rows32-d128", False, 6, 8, 2, 128, 128, 16, (257, 640), 16), ("rows32-d64", False, 31, 4, 4, 64, 64, 64, (480, 90), 16),
    ("rows64-d128", False, 8, 16, 2, 128, 128, 64, (333, 900), 16), ("rows64-d64", False, 16, 8, 2, 64, 64, 32, (450, 60), 16),
    ("rows16-d128-e4m3", True, 1, 8, 2, 128, 128, 64, (300, 77), 16), ("rows32-d64-e4m3", True, 6, 8, 2, 64, 64, 16, (511, 30), 16),
    ("rows64-d128-e4m3", True, 8, 16, 2, 128, 128, 64, (333, 900), 16), ("ranges-d128", False, 1, 8, 2, 128, 128, 64, (2500,), 16),
    ("d96", False, 5, 8, 2, 96, 40, 16, (300, 50), None), ("d96-e4m3", True, 40, 4, 2, 96, 80, 64, (300, 50), None),
    ("d192", False, 5, 8, 2, 192, 128, 16, (300, 50), None), ("odd", False, 3, 4, 2, 33, 31, 8, (300, 50), None)]


def _once(c):
    """out of the float64 formula with exp(s - max) rounded to bfloat16 before the product with v."""
    q, k, v = (c[n].double().cpu() for n in "qkv") if c["ks"] is None else (
        c["q"].double().cpu(), ref.values(c["k"], c["ks"]).cpu(), ref.values(c["v"], c["vs"]).cpu())
    B, S, Hq, D = q.shape
    G, ps, bt = Hq // k.shape[2], k.shape[1], c["bt"].cpu()
    out = torch.zeros(B, S, Hq, v.shape[3], dtype=torch.float64)
    for b, ctx in enumerate(c["ctx"].tolist()):
        at = torch.arange(ctx + S)
        pg = bt[b, at // ps].long()
        ok = ref.seen(ctx + torch.arange(S), ctx + S, None, 0)
        for h in range(Hq):
            z = (q[b, :, h] @ k[pg, at % ps, h // G].t() / math.sqrt(D)).masked_fill(~ok, -math.inf)
            p = torch.exp(z - z.amax(1, keepdim=True))
            out[b, :, h] = p.float().to(BF).double() @ v[pg, at % ps, h // G] / p.sum(1, keepdim=True)
    return out.to(BF).double()


@pytest.mark.parametrize("case", CASES, ids=[c[0] for c in CASES])
def test_weights_keep_their_bits(case):
    _, fp8, S, Hq, Hkv, D, Dv, page, ctx, bits = case
    c = _case(BF, fp8, S=S, ctx=ctx, Hq=Hq, Hkv=Hkv, D=D, Dv=Dv, page=page, seed=61)
    c["q"] *= 0.5
    w = 0.0 if bits is None else 2.0 ** -bits
    want = _want(c)
    ref.check(_run(c), want, D, BF, w)
    o, _, pv, mag, num = (x.cpu() for x in want)
    bound = ref.half(BF) * o.abs() * (1 + w) + (ref.row_error(D, mag, num)[..., None] + w) * pv
    # (over 2500 keys the sums' own bound, (1.25 * 2500 + 64) 2^-24 = 2^-12.4, is more than the
    # 2^-9 / sqrt(2500) = 2^-14.6 that the keys' roundings to one part come to: there one part passes)
    assert max(ctx) > 1000 or bool(((_once(c) - o).abs() > bound).any())


@pytest.mark.parametrize("S,heads,D,Dv,w", [(16, (8, 2), 64, 64, 2.0 ** -16), (40, (4, 4), 128, 128, 2.0 ** -16), (150, (8, 2), 96, 96, 0.0),
                                            (200, (4, 1), 40, 24, 0.0), (150, (8, 2), 192, 160, 0.0)])
def test_whole_sequences(S, heads, D, Dv, w):
    q, k, v, _, sink = _leaves(BF, B=2, S=S, Hq=heads[0], Hkv=heads[1], D=D, Dv=Dv)
    bt = torch.arange(2, device=DEV, dtype=torch.int32).view(2, 1)
    ctx = torch.zeros(2, device=DEV, dtype=torch.int32)
    pool = [torch.cat((t, t.new_zeros(2, 256 - S, *t.shape[2:])), 1) for t in (k, v)]
    ref.check(ops_amd.window_attention(q, k, v, attn_sink=sink), ref.chunk(q, *pool, bt, ctx, None, sink=sink), D, BF, w)


@pytest.mark.parametrize("D,Dv", [(96, 96), (40, 24), (33, 7), (192, 160), (300, 300)])
def test_gradients_of_other_dims_keep_float32_weights(D, Dv):
    """p and ds are not rounded: only o (in delta) and the results are bfloat16."""
    x = _leaves(BF, B=2, S=200, Hq=8, Hkv=2, D=D, Dv=Dv)
    lens = torch.tensor([200, 77], dtype=torch.int32, device=DEV)
    got = _run_window(*x, lens=lens, window=90, first=3)
    ref.check_all(got, ref.window(*x[:4], lens, 90, 3, x[4], None, None, BF, 0.0))
