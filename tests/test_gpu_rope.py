"""GPU tests of the rotation and the per-head norms (forward, backward, append
into pages) against float64.

Tolerances: a result rounded to its type is off by at most finfo.eps / 2 of its
value.  Before that everything is float32: u = x r w carries at most 8
roundings, sin and cos 2 ulp each, the products and the sum 3 more, all
relative to the pair's length M = |(u1, u2)|, hence 2^-20 M.  dx = r (g - xhat m)
adds sums over a row (at most 14 roundings deep): 2^-18 of the magnitudes that
enter it.  dw sums N rows, at most N / 1024 + 40 additions deep."""
import math

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


def _randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def _half(dt):
    return torch.finfo(dt).eps / 2


def _pair_len(u, off, R, interleaved):
    """Per element: the length of its rotated pair, or its own size."""
    m = u.abs().clone()
    p = u[..., off:off + R]
    if interleaved:
        n = (p[..., 0::2].square() + p[..., 1::2].square()).sqrt().repeat_interleave(2, -1)
    else:
        n = (p[..., :R // 2].square() + p[..., R // 2:].square()).sqrt().repeat(1, 1, 1, 2)
    m[..., off:off + R] = n
    return m


def _close(got, want, bound, what):
    bad = (got.double() - want).abs() - bound
    assert torch.isfinite(got.double()).all(), what
    assert float(bad.max()) <= 0.0, (what, float(bad.max()), float((got.double() - want).abs().max()))


def _fwd_ref(x, w, pos, freq, eps, off, inter, scale):
    u, h, r = ref.norm(x.double(), w, eps)
    y = ref.rotate(u, pos, freq, off, inter, scale)
    return y, _pair_len(u, off, 2 * freq.numel(), inter) * max(1.0, abs(scale)), h, r


def _bwd_ref(dy, x, w, pos, freq, eps, off, inter, scale):
    """dx, its bound's magnitude, dw, its magnitude."""
    du = ref.rotate(dy.double(), pos, freq, off, inter, scale, back=True)
    dm = _pair_len(dy.double(), off, 2 * freq.numel(), inter) * max(1.0, abs(scale))
    if w is None:
        return du, dm, None, None
    n = w.numel()
    _, h, r = ref.norm(x.double(), w, eps)
    wd = w.double()
    g = du[..., :n] * wd
    m = (g * h).mean(-1, keepdim=True)
    mm = (dm[..., :n] * wd.abs() * h.abs()).mean(-1, keepdim=True)
    dx, mag = du.clone(), dm.clone()
    dx[..., :n] = r * (g - h * m)
    mag[..., :n] = r * (dm[..., :n] * wd.abs() + h.abs() * mm)
    t = du[..., :n] * h
    return dx, mag, t.reshape(-1, n).sum(0), (dm[..., :n] * h.abs()).reshape(-1, n).sum(0)


CASES = [
    # B, S, Hq, Hkv, D, R, off, interleaved, q norm, k norm, dtype, weight dtype
    (1, 1, 1, 1, 64, 64, 0, False, 64, 64, BF16, BF16),
    (2, 33, 8, 2, 128, 128, 0, False, 128, 128, BF16, BF16),
    (2, 33, 8, 2, 128, 128, 0, True, 128, 128, BF16, F32),
    (3, 17, 5, 3, 64, 32, 0, False, 64, 64, F32, F32),
    (1, 9, 7, 1, 64, 32, 32, True, 64, 0, BF16, BF16),
    (2, 5, 16, 1, 576, 64, 512, True, 0, 512, BF16, BF16),   # latent rows
    (1, 6, 3, 1, 576, 64, 512, False, 512, 512, BF16, F32),
    (1, 7, 2, 2, 192, 64, 128, False, 192, 128, BF16, BF16),  # 24 chunks on 32 lanes
    (1, 4, 2, 1, 1024, 1024, 0, False, 1024, 1024, F32, F32),
    (1, 4, 2, 1, 1024, 512, 256, True, 512, 1024, BF16, BF16),
    (1, 3, 2, 1, 288, 96, 96, False, 288, 192, F32, F32),     # 72 float32 chunks
    (2, 11, 3, 1, 80, 40, 0, False, 80, 80, BF16, BF16),      # half the rotation is not whole chunks
    (2, 11, 3, 1, 77, 30, 3, True, 50, 77, F32, F32),         # odd sizes throughout
    (1, 5, 2, 1, 33, 2, 31, False, 0, 33, BF16, BF16),
    (1, 1500, 4, 2, 128, 128, 0, False, 128, 128, BF16, BF16),
]


def _inputs(c, seed=0, pos0=0):
    B, S, Hq, Hkv, D, R, off, inter, nq, nk, dt, wt = c
    g = _g(seed)
    q, k = _randn(g, B, S, Hq, D, dtype=dt), _randn(g, B, S, Hkv, D, dtype=dt)
    wq = (1 + 0.2 * _randn(g, nq)).to(wt) if nq else None
    wk = (1 + 0.2 * _randn(g, nk)).to(wt) if nk else None
    pos = torch.randint(0, 4096, (B, S), generator=g, device=DEV) + pos0
    return q, k, wq, wk, pos, ops_amd.rope_frequencies(R, device=DEV)


@pytest.mark.parametrize("c", CASES, ids=[f"D{c[4]}R{c[5]}o{c[6]}{'i' if c[7] else 'h'}n{c[8]}-{c[9]}{str(c[10])[6:]}"
                                          for c in CASES])
def test_norm_rope_forward_backward(c):
    off, inter, dt, wt = c[6], c[7], c[10], c[11]
    q, k, wq, wk, pos, freq = _inputs(c)
    leaves = [t if t is None else t.requires_grad_(True) for t in (q, k, wq, wk)]
    yq, yk = ops_amd.qk_norm_rope(q, k, pos, freq, wq, wk, eps=1e-5, rope_offset=off, interleaved=inter, rope_scale=1.25)
    g = _g(7)
    dq, dk = _randn(g, *q.shape, dtype=dt), _randn(g, *k.shape, dtype=dt)
    grads = torch.autograd.grad([yq, yk], [t for t in leaves if t is not None], [dq, dk])
    torch.cuda.synchronize()
    dws = list(grads[2:])
    for name, x, w, y, dy, dx in (("q", q, wq, yq, dq, grads[0]), ("k", k, wk, yk, dk, grads[1])):
        x, w = x.detach(), None if w is None else w.detach()
        want, mag, _, _ = _fwd_ref(x, w, pos, freq, 1e-5, off, inter, 1.25)
        assert y.dtype == dt and y.shape == x.shape
        _close(y.detach(), want, _half(dt) * want.abs() + 2.0 ** -20 * mag, name)
        wdx, mag, wdw, wmag = _bwd_ref(dy, x, w, pos, freq, 1e-5, off, inter, 1.25)
        _close(dx, wdx, _half(dt) * wdx.abs() + 2.0 ** -18 * mag, "d" + name)
        if w is not None:
            dw = dws.pop(0)
            n = x[..., 0].numel()
            assert dw.dtype == wt and dw.shape == w.shape
            _close(dw, wdw, _half(wt) * wdw.abs() + (2.0 ** -19 + (n / 1024 + 40) * 2.0 ** -24) * wmag, "dw" + name)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("pos0,i64", [(0, False), (1 << 20, True), ((1 << 31) - 8192, False), (-5000, True)])
def test_rotary_far_positions(dt, pos0, i64):
    g = _g(3)
    x = _randn(g, 2, 6, 3, 128, dtype=dt)
    pos = (pos0 + torch.randint(0, 4096, (2, 6), generator=g, device=DEV)).to(torch.int64 if i64 else torch.int32)
    freq = ops_amd.rope_frequencies(128, scaling="ntk", factor=8.0, device=DEV)
    y = ops_amd.rotary_embedding(x, pos, freq)
    want = ref.rotate(x.double(), pos, freq, 0, False)
    mag = _pair_len(x.double(), 0, 128, False)
    # pos f in float64 is itself off by 2^-52 of the angle, on both sides
    far = (pos.double().abs().max() * 2.0 ** -51) * mag
    _close(y, want, _half(dt) * want.abs() + 2.0 ** -20 * mag + far, "y")


def test_rotary_gradient_against_differences():
    """In float32 the rotation is linear: (f(x + e) - f(x)) . dy = e . dx."""
    g = _g(4)
    x = _randn(g, 1, 7, 2, 64).requires_grad_(True)
    w = (1 + 0.1 * _randn(g, 64)).requires_grad_(True)
    k = _randn(g, 1, 7, 1, 64)
    pos, freq = torch.arange(7, device=DEV), ops_amd.rope_frequencies(64, device=DEV)
    dy = _randn(g, 1, 7, 2, 64)

    def f(xx, ww):
        with torch.no_grad():
            u, _, _ = ref.norm(xx.double(), ww.double(), 1e-6)
            return float((ref.rotate(u, pos[None], freq, 0, False) * dy.double()).sum())

    y, _ = ops_amd.qk_norm_rope(x, k, pos, freq, w, None)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    for leaf, grad in ((x, dx), (w, dw)):
        e = torch.randn(leaf.shape, generator=g, device=DEV, dtype=torch.float64)
        h = 1e-4
        xp = (leaf.detach().double() + h * e, leaf.detach().double() - h * e)
        d = [(f(v, w.detach()) if leaf is x else f(x.detach(), v)) for v in xp]
        num = (d[0] - d[1]) / (2 * h)
        # central differences: h^2 of the third derivative, of the order of the gradient's size
        size = float((grad.double().abs() * e.abs()).sum())
        assert abs(num - float((grad.double() * e).sum())) <= 1e-4 * size


def test_rotary_strided_view_out_and_in_place():
    g = _g(5)
    base = _randn(g, 2, 9, 4, 576, dtype=BF16)
    keep = base.clone()
    pos, freq = torch.arange(9, device=DEV, dtype=torch.int32), ops_amd.rope_frequencies(64, device=DEV)
    want = ops_amd.rotary_embedding(base[..., 512:], pos, freq, interleaved=True)
    ops_amd.rotary_embedding(base[..., 512:], pos, freq, interleaved=True, out=base[..., 512:])
    assert torch.equal(base[..., 512:], want) and torch.equal(base[..., :512], keep[..., :512])
    # rows whose parts pair across lanes and chunks, in place: vector and scalar kernels
    for D, R, off in ((128, 128, 0), (576, 576, 0), (80, 40, 0), (1024, 1024, 0)):
        x = _randn(g, 1, 5, 3, D, dtype=BF16)
        f = ops_amd.rope_frequencies(R, device=DEV)
        p = torch.arange(5, device=DEV)
        want = ops_amd.rotary_embedding(x, p, f, rope_offset=off)
        assert torch.equal(ops_amd.rotary_embedding(x, p, f, rope_offset=off, out=x), want)


def test_one_sided_gradients_and_empty():
    g = _g(6)
    q, k = _randn(g, 1, 4, 2, 64).requires_grad_(True), _randn(g, 1, 4, 1, 64).requires_grad_(True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    pos, freq = torch.arange(4, device=DEV), ops_amd.rope_frequencies(64, device=DEV)
    y, z = ops_amd.qk_norm_rope(q, k, pos, freq, w, w)
    z.sum().backward()
    assert q.grad is None and k.grad is not None and w.grad is not None
    only_k = w.grad.clone()
    y, z = ops_amd.qk_norm_rope(q, k, pos, freq, w, w)
    (y.sum() + z.sum()).backward()   # one weight for both: its gradients add up
    assert not torch.equal(w.grad, 2 * only_k)
    e = torch.empty(0, 4, 2, 64, device=DEV, requires_grad=True)
    ye, ze = ops_amd.qk_norm_rope(e, e, pos, freq, w, None)
    de, dwe = torch.autograd.grad(ye.sum() + ze.sum(), [e, w])
    assert ye.shape == e.shape and de.shape == e.shape and float(dwe.abs().sum()) == 0.0


def test_zero_rows_have_finite_results():
    x = torch.zeros(1, 3, 2, 128, device=DEV, dtype=BF16, requires_grad=True)
    w = torch.ones(128, device=DEV, dtype=BF16, requires_grad=True)
    pos, freq = torch.arange(3, device=DEV), ops_amd.rope_frequencies(128, device=DEV)
    y, _ = ops_amd.qk_norm_rope(x, x.detach(), pos, freq, w, None)
    dx, dw = torch.autograd.grad(y.float().sum(), [x, w])
    assert float(y.abs().max()) == 0.0 and torch.isfinite(dx).all() and float(dw.abs().max()) == 0.0


@pytest.mark.parametrize("D,Dv,Hq,Hkv,off,R,nk,inter,dt", [
    (128, 128, 8, 2, 0, 128, 128, False, BF16), (576, 0, 16, 1, 512, 64, 512, True, BF16),
    (64, 128, 4, 4, 0, 32, 0, False, F32), (77, 33, 3, 3, 5, 30, 77, False, BF16)])
@pytest.mark.parametrize("S", [1, 13])
def test_append(D, Dv, Hq, Hkv, off, R, nk, inter, dt, S):
    """k rows equal qk_norm_rope's bit for bit, v rows are copied, and nothing
    else in the pool changes; padded tokens and unmapped pages are left out."""
    g = _g(8)
    B, ps, npages = 3, 8, 20
    q, k = _randn(g, B, S, Hq, D, dtype=dt), _randn(g, B, S, Hkv, D, dtype=dt)
    v = _randn(g, B, S, Hkv, Dv, dtype=dt) if Dv else None
    wk = (1 + 0.2 * _randn(g, nk)).to(dt) if nk else None
    kc = _randn(g, npages, ps, Hkv, D, dtype=dt)
    vc = _randn(g, npages, ps, Hkv, Dv, dtype=dt) if Dv else None
    bt = torch.randperm(npages, generator=g, device=DEV)[:18].view(3, 6).to(torch.int32)
    bt[2, 1] = -1
    bt[1, 0] = npages  # outside the pool
    slots = (torch.arange(S, device=DEV) + 5).expand(B, S).clone()
    slots[0, 0] = -1
    slots[2, -1] = 6 * ps  # outside the table
    pos = torch.randint(0, 100, (B, S), generator=g, device=DEV)
    freq = ops_amd.rope_frequencies(R, device=DEV)
    kc0, vc0 = kc.clone(), None if vc is None else vc.clone()
    wq, wkk = ops_amd.qk_norm_rope(q, k, pos, freq, None, wk, rope_offset=off, interleaved=inter)
    out = ops_amd.qk_norm_rope_append(q, k, v, kc, vc, bt, slots, pos, freq, None, wk, rope_offset=off, interleaved=inter)
    torch.cuda.synchronize()
    assert torch.equal(out, wq)
    for b in range(B):
        for s in range(S):
            e = int(slots[b, s])
            if not 0 <= e < 6 * ps or not 0 <= int(bt[b, e // ps]) < npages:
                continue
            kc0[int(bt[b, e // ps]), e % ps] = wkk[b, s]
            if vc is not None:
                vc0[int(bt[b, e // ps]), e % ps] = v[b, s]
    assert torch.equal(kc, kc0) and (vc is None or torch.equal(vc, vc0))


def test_append_far_into_a_large_pool():
    """Row offsets past 2^31 elements."""
    D, ps = 576, 64
    npages = (1 << 31) // (ps * D) + 8
    kc = torch.zeros(npages, ps, 1, D, dtype=BF16, device=DEV)
    k = _randn(_g(9), 1, 2, 1, D, dtype=BF16)
    bt = torch.tensor([[0, npages - 1]], dtype=torch.int32, device=DEV)
    slots = torch.tensor([[3, 2 * ps - 1]], device=DEV)
    freq = ops_amd.rope_frequencies(64, device=DEV)
    ops_amd.qk_norm_rope_append(None, k, None, kc, None, bt, slots, slots, freq, rope_offset=512)
    want = ops_amd.rotary_embedding(k, slots, freq, rope_offset=512)
    assert torch.equal(kc[0, 3], want[0, 0]) and torch.equal(kc[npages - 1, ps - 1], want[0, 1])
    assert int((kc[1:-1] != 0).sum()) == 0


def test_captured_step_and_other_stream():
    g = _g(10)
    q, k = _randn(g, 1, 64, 4, 128, dtype=BF16).requires_grad_(True), _randn(g, 1, 64, 2, 128, dtype=BF16).requires_grad_(True)
    w = torch.ones(128, device=DEV, dtype=BF16).requires_grad_(True)
    dq, dk = _randn(g, 1, 64, 4, 128, dtype=BF16), _randn(g, 1, 64, 2, 128, dtype=BF16)
    pos, freq = torch.arange(64, device=DEV), ops_amd.rope_frequencies(128, device=DEV)

    def step():
        y, z = ops_amd.qk_norm_rope(q, k, pos, freq, w, w)
        return [y.detach(), z.detach(), *torch.autograd.grad([y, z], [q, k, w], [dq, dk])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(_randn(_g(20 + i), 1, 64, 4, 128, dtype=BF16))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    assert all(torch.isfinite(t).all() for t in on_side)


def test_backward_is_deterministic():
    c = (2, 300, 8, 2, 128, 128, 0, False, 128, 128, BF16, F32)
    q, k, wq, wk, pos, freq = _inputs(c, seed=11)
    for t in (q, k, wq, wk):
        t.requires_grad_(True)
    runs = []
    for _ in range(2):
        y, z = ops_amd.qk_norm_rope(q, k, pos, freq, wq, wk)
        runs.append(torch.autograd.grad([y, z], [q, k, wq, wk], [torch.ones_like(y), torch.ones_like(z)]))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
