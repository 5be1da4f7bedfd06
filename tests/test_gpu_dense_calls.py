"""Dense attention as programs call it: graphs, streams, caches beyond 32-bit offsets,
padding left alone, and the operators one after another."""
import math

import pytest
import torch

import ops_amd
from tests import dense_ref as ref
from tests.test_gpu_dense import BF, DEV, F32, _case, _run, _want
from tests.test_gpu_window import _check, _leaves
from tests.test_gpu_window import _run as _run_window

pytestmark = pytest.mark.gpu

CASES = {
    "decode": dict(S=1, ctx=(40, 900), Hq=8, Hkv=2, D=128, page=64),
    "chunk": dict(S=90, ctx=(40, 700), Hq=8, Hkv=2, D=64, page=16),
    "e4m3": dict(S=1, ctx=(300, 2000), Hq=8, Hkv=1, D=128, page=64, fp8=True),
    "latent": dict(S=3, ctx=(300, 64), Hq=16, Hkv=1, D=576, Dv=512, mla=True, page=64),
    "f32": dict(dtype=F32, S=5, ctx=(100, 30), Hq=4, Hkv=2, D=96, page=16),
}


def _eager_work():
    x = torch.randn(512, 512, device=DEV)
    for _ in range(3):
        x = torch.tanh(x @ x)
    torch.cuda.synchronize()


@pytest.mark.parametrize("names", [("decode", "e4m3"), ("chunk", "latent"), ("f32", "decode")])
def test_captured_calls_follow_their_inputs(names):
    """Two graphs at a time, replayed in turn with new inputs in place."""
    graphs = []
    for i, name in enumerate(names):
        c = _case(seed=i, **CASES[name])
        out, lse = (t.clone() for t in _run(c))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = _run(c)
        graphs.append((c, g, res, out, lse))
    for k in range(4):
        for c, g, res, out, lse in graphs:
            if k == 2:  # shorter contexts, other queries
                c["ctx"].sub_(7)
                c["q"].mul_(0.5)
                out, lse = _run(c)
            elif k > 2:
                out, lse = _run(c)
            g.replay()
            _eager_work()
            assert torch.equal(res[0], out) and torch.equal(res[1], lse), k


@pytest.mark.parametrize("dtype,S", [(BF, 300), (F32, 130)])
def test_captured_training_step(dtype, S):
    x = _leaves(dtype, B=2, S=S, Hq=8, Hkv=2, D=64)
    lens = torch.tensor([S, S - 40], dtype=torch.int32, device=DEV)

    def step():
        xs = [t.detach().requires_grad_(True) for t in (x[0], x[1], x[2], x[4])]
        out, lse = ops_amd.window_attention(*xs[:3], window=100, first=3, lens=lens, attn_sink=xs[3])
        return [out.detach(), lse.detach(), *torch.autograd.grad(out, xs, x[3])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = step()
    for k in range(4):
        if k == 2:
            x[0].mul_(0.5)
            lens.sub_(17)
        want = [t.clone() for t in step()]
        g.replay()
        _eager_work()
        assert all(torch.equal(a, b) for a, b in zip(res, want)), k


@pytest.mark.parametrize("name", list(CASES))
def test_another_stream(name):
    c = _case(**CASES[name])
    want = _run(c)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        q = c["q"].clone()
        big = torch.randn(2048, 2048, device=DEV)
        for _ in range(20):
            big = torch.tanh(big @ big)
        c["q"] = q.copy_(q + 0 * big[0, 0].to(q.dtype))  # (ready only after the products)
        got = _run(c)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", [1, 40])
def test_rows_of_no_scale(S, D):
    """Exponent byte 255: NaN for the tokens that see the row, nothing for the others."""
    c = _case(fp8=True, S=S, ctx=(200, 100), Hq=8, Hkv=2, D=D, page=64)
    want = _run(c)
    j = 50
    pg = int(c["bt"][0, j // 64])
    for scales in ("ks", "vs"):
        old = int(c[scales][pg, j % 64, 1])
        c[scales][pg, j % 64, 1] = 255
        out, lse = _run(c)
        assert torch.equal(out[1], want[0][1]) and torch.equal(out[0, :, :4], want[0][0, :, :4])
        assert torch.isnan(out[0, :, 4:]).all()
        assert torch.isnan(lse[0, :, 4:]).all() == (scales == "ks")
        win = _run(c, window=40)
        c[scales][pg, j % 64, 1] = old
        again = _run(c, window=40)
        assert torch.equal(win[0], again[0]) and torch.equal(win[1], again[1])


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "latent"])
def test_caches_beyond_32_bit_offsets(kind):
    """Pools of more than 2^32 bytes (and 2^31 elements), the sequences' pages at both ends."""
    fp8, mla = kind == "e4m3", kind == "latent"
    kw = dict(S=2, ctx=(150, 70), page=64, fp8=fp8)
    kw.update(dict(Hq=16, Hkv=1, D=576, Dv=512, mla=True) if mla else dict(Hq=8, Hkv=4, D=128))
    c = _case(**kw)
    want = _run(c)
    num = c["k"].shape[0]
    rows = c["k"][0].numel()
    total = (1 << 32) // rows + num + 5

    def spread(t):
        big = torch.empty(total, *t.shape[1:], dtype=torch.uint8 if t.element_size() == 1 else t.dtype, device=DEV)
        big[:2].copy_(t.view(big.dtype)[:2])
        big[-(num - 2):].copy_(t.view(big.dtype)[2:])
        return big.view(t.dtype)
    for name in ("k", "ks", "vs") if mla else ("k", "v", "ks", "vs"):
        if c[name] is not None:
            c[name] = spread(c[name])
    if mla:
        c["v"] = c["k"][..., :512]
    ok = (c["bt"] >= 2) & (c["bt"] < num)
    c["bt"] = torch.where(ok, c["bt"] + (total - num), c["bt"])
    got = _run(c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype,S,heads,D,window", [
    (BF, 1500, (8, 1), 128, None), (BF, 1500, (8, 1), 64, 300), (BF, 700, (32, 2), 128, 1), (F32, 700, (16, 1), 64, None),
    (F32, 500, (12, 1), 96, 130), (F32, 400, (8, 1), 160, None), (BF, 400, (8, 1), 40, 70),
])
def test_key_blocks_cut_in_chunks(dtype, S, heads, D, window):
    """Few key blocks that many rows see: their sums are of several workgroups."""
    _check(_leaves(dtype, B=1, S=S, Hq=heads[0], Hkv=heads[1], D=D), window=window, first=5 if window else 0)


def test_more_key_blocks_than_are_sorted():
    """A window of one: a token's result is its own v, its gradients are do for v and zero for q and
    k (the only weight is 1), exactly; blocks of 128 keys, some rows padded."""
    S, n = 4096 * 128 + 300, 4096 * 128 + 171
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v, do = (torch.randn(1, S, 1, 64, generator=g, device=DEV).to(BF) for _ in range(4))
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    xs = [t.requires_grad_(True) for t in (q, k, v)]
    out, _ = ops_amd.window_attention(*xs, window=1, lens=lens)
    dq, dk, dv = torch.autograd.grad(out, xs, do)
    assert torch.equal(out[:, :n], v[:, :n]) and torch.equal(dv[:, :n], do[:, :n])
    assert not out[:, n:].any() and not dv[:, n:].any() and not dq[:, n:].any() and not dk[:, n:].any()
    # (ds = do.v - do.o: 64 products of float32 in two orders, times a row of up to 6)
    mag = (do.float() * v.detach().float()).abs().sum(-1).max()
    assert float(torch.stack((dq, dk)).abs().max()) <= 128 * 2.0 ** -24 * float(mag) * 6


@pytest.mark.parametrize("D,Dv,S", [(64, 64, 300), (128, 128, 200), (96, 96, 150), (192, 160, 90)])
def test_the_sinks_gradient_knows_no_bf16(D, Dv, S):
    """A float32 sum over all rows: as if o had not been rounded to bf16 (and with float32's bounds)."""
    x = _leaves(BF, B=2, S=S, Hq=8, Hkv=2, D=D, Dv=Dv)
    dlse = torch.randn(2, S, 8, device=DEV)
    for grad in (None, dlse):
        got = _run_window(*x, dlse=grad, window=70, first=3)
        want, bound = ref.window(*x[:4], None, 70, 3, x[4], grad, None, F32, 0.0)[5]
        assert float(((got[5].double() - want).abs() - bound).max()) <= 0.0


def test_padded_rows_in_chunks():
    x = _leaves(F32, B=2, S=600, Hq=8, Hkv=1, D=64)
    lens = torch.tensor([600, 33], dtype=torch.int32, device=DEV)
    got = _check(x, lens=lens)
    for t in got[3:5]:
        assert not t[1, 33:].any()


def test_what_is_behind_the_last_row_stays():
    """Only rows of the tensors are written: not the memory around them."""
    c = _case(S=5, ctx=(40, 70), Hq=8, Hkv=2, D=64)
    whole = torch.full((2, 9, 10, 64), 7.0, device=DEV, dtype=BF)
    lse = torch.full((2, 9, 10), 7.0, device=DEV)
    got = _run(c, out=whole[:, 2:7, 1:9], lse=lse[:, 2:7, 1:9])
    want = _run(c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for t in (whole, lse):
        t[:, 2:7, 1:9] = 7.0
        assert bool((t == 7.0).all())


def test_a_layer_trained():
    """q and k normalised and rotated, attended to through a window, all gradients, against float64."""
    B, S, Hq, Hkv, D, window = 2, 90, 8, 2, 64, 33
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = (torch.randn(B, S, h, D, generator=g, device=DEV) for h in (Hq, Hkv, Hkv))
    wq, wk = (1.0 + 0.1 * torch.randn(D, generator=g, device=DEV) for _ in range(2))
    do = torch.randn(B, S, Hq, D, generator=g, device=DEV)
    pos = torch.arange(S, device=DEV, dtype=torch.int32)
    ang = pos.double()[:, None] * torch.pow(10000.0, -torch.arange(0, D, 2, device=DEV).double() / D)
    cos, sin = ang.cos(), ang.sin()

    def normed(x, w, rot):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        c, s = (t.to(x.dtype)[:, None, :] for t in rot)
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    def plain():
        xs = [t.double().requires_grad_(True) for t in (q, k, v, wq, wk)]
        a, b = normed(xs[0], xs[3], (cos, sin)), normed(xs[1], xs[4], (cos, sin))
        s = torch.einsum("bshd,bthd->bhst", a, b.repeat_interleave(Hq // Hkv, 2)) / math.sqrt(D)
        p = torch.softmax(s.masked_fill(~ref.seen(pos, S, window, 2), -math.inf), -1)
        o = torch.einsum("bhst,bthd->bshd", p, xs[2].repeat_interleave(Hq // Hkv, 2))
        return [o.detach(), *torch.autograd.grad(o, xs, do.double())]

    xs = [t.clone().requires_grad_(True) for t in (q, k, v, wq, wk)]
    a, b = normed(xs[0], xs[3], (cos, sin)), normed(xs[1], xs[4], (cos, sin))
    o, _ = ops_amd.window_attention(a, b, xs[2], window=window, first=2)
    for x, y in zip([o.detach(), *torch.autograd.grad(o, xs, do)], plain()):
        # (float32 throughout: a few hundred roundings of the largest value)
        assert float((x.double() - y).abs().max()) <= 400 * 2.0 ** -24 * float(y.abs().max())
