"""Causal attention of whole sequences through a window, forward and backward,
against float64 (tests/dense_ref.py derives the tolerances)."""
import math

import pytest
import torch

import ops_amd
from tests import dense_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
types = pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])


def _leaves(dtype, B=2, S=70, Hq=4, Hkv=2, D=64, Dv=None, seed=0, sink=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    Dv = D if Dv is None else Dv

    def r(*s):
        return torch.randn(s, generator=g, device=DEV).to(dtype)
    q, k, v, do = 2.0 * r(B, S, Hq, D), r(B, S, Hkv, D), r(B, S, Hkv, Dv), r(B, S, Hq, Dv)
    sk = torch.randn(Hq, generator=g, device=DEV) if sink else None
    return q, k, v, do, sk


def _run(q, k, v, do, sink, lens=None, dlse=None, **kw):
    xs = [t.detach().requires_grad_(True) for t in (q, k, v, sink) if t is not None]
    out, lse = ops_amd.window_attention(*xs[:3], lens=lens, attn_sink=xs[3] if sink is not None else None, **kw)
    if dlse is None:
        grads = torch.autograd.grad(out, xs, do)
    else:
        grads = torch.autograd.grad([out, lse], xs, [do, dlse])
    return [out.detach(), lse.detach(), *grads]


def _check(x, lens=None, dlse=None, window=None, first=0, sm_scale=None):
    q, k, v, do, sink = x
    got = _run(*x, lens=lens, dlse=dlse, window=window, first=first, sm_scale=sm_scale)
    ref.check_all(got, ref.window(q, k, v, do, lens, window, first, sink, dlse, sm_scale, q.dtype, 2.0 ** -8 if q.dtype == BF else 0.0))
    return got


@types
@pytest.mark.parametrize("D,Dv", [(64, 64), (128, 128), (96, 40), (33, 7), (192, 128), (300, 20)])
def test_head_dims(dtype, D, Dv):
    _check(_leaves(dtype, D=D, Dv=Dv))


@types
@pytest.mark.parametrize("S", [1, 2, 33, 64, 129, 300])
@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (16, 1), (10, 2)])
def test_lengths_and_heads(dtype, S, heads):
    _check(_leaves(dtype, B=1, S=S, Hq=heads[0], Hkv=heads[1], D=128 if S % 2 else 64, seed=S, sink=S != 64))


@types
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 2), (17, 0), (64, 4), (65, 64), (130, 200), (None, 9), (5, 1 << 30)])
def test_windows(dtype, D, window, first):
    _check(_leaves(dtype, B=1, S=290, D=D), window=window, first=first)


@types
def test_padded_batches(dtype):
    """Padding is not read (NaN), gives zeros and -inf and gets zero gradients."""
    B, S = 5, 150
    lens = [150, 0, 1, 77, 64]
    for D in (64, 128):
        q, k, v, do, sink = _leaves(dtype, B=B, S=S, D=D, Hq=8)
        for b, n in enumerate(lens):
            for t in (q, k, v, do):
                t[b, n:] = math.nan
        for type_ in (torch.int32, torch.int64):
            n = torch.tensor(lens, dtype=type_, device=DEV)
            for kw in (dict(), dict(window=20, first=3)):
                got = _check((q.nan_to_num(), k.nan_to_num(), v.nan_to_num(), do.nan_to_num(), sink), n, **kw)
                same = _run(q, k, v, do, sink, n, **kw)
                assert all(torch.equal(a, b) for a, b in zip(got, same))
                for x in (got[0], got[2], got[3], got[4]):
                    assert all(float(x[b, m:].abs().sum()) == 0.0 for b, m in enumerate(lens))


@types
def test_gradient_of_the_lse(dtype):
    x = _leaves(dtype, S=100)
    dlse = torch.randn(2, 100, 4, device=DEV)
    _check(x, dlse=dlse, window=40)
    q, k, v, do, sink = x
    lse = ops_amd.window_attention(q.requires_grad_(True), k, v)[1]
    dq = torch.autograd.grad(lse, q, dlse)[0]
    want = ref.window(q.detach(), k, v, torch.zeros_like(do), None, None, 0, None, dlse, None, dtype, 2.0 ** -8)[2]
    assert float(((dq.double() - want[0]).abs() - want[1]).max()) <= 0.0


def test_formula_against_differences():
    """The float64 formula that the kernels are held to, by central differences."""
    torch.manual_seed(0)
    q, k, v, do = (torch.randn(1, 9, h, 4, dtype=torch.float64) for h in (2, 1, 1, 2))
    sink, dlse = torch.randn(2, dtype=torch.float64), torch.randn(1, 9, 2, dtype=torch.float64)

    def loss(q, k, v, sink):
        r = ref.window(q, k, v, do, None, 4, 2, sink, dlse)
        return float((r[0][0] * do).sum() + (r[1][0] * dlse).sum())
    grads = [g for g, _ in ref.window(q, k, v, do, None, 4, 2, sink, dlse)[2:]]
    xs, eps = [q, k, v, sink], 1e-5
    for i, (x, g) in enumerate(zip(xs, grads)):
        for at in range(0, x.numel(), 3):
            d = torch.zeros_like(x).view(-1)
            d[at] = eps
            up, dn = ([y + s * d.view(x.shape) if j == i else y for j, y in enumerate(xs)] for s in (1, -1))
            # (third derivatives of order 10 at 1e-5: 1e-9, and 1e-16 / 1e-5 of rounding)
            assert abs((loss(*up) - loss(*dn)) / (2 * eps) - float(g.view(-1)[at])) < 1e-7


@types
def test_kernels_against_differences(dtype):
    """Along random directions, the float64 formula's change against the kernels' gradients
    within their bounds."""
    x = _leaves(dtype, B=1, S=80, D=128)
    q, k, v, do, sink = x
    got = _run(*x, window=30, first=2)
    want = ref.window(q, k, v, do, None, 30, 2, sink, None, None, dtype, 2.0 ** -8 if dtype == BF else 0.0)
    for i, t in enumerate((q, k, v, sink)):
        d = torch.randn_like(t.double())
        at = [y.double() for y in (q, k, v, sink)]

        def loss(s):
            z = [y + s * d if j == i else y for j, y in enumerate(at)]
            return float((ref.window(*z[:3], do.double(), None, 30, 2, z[3])[0][0] * do.double()).sum())
        diff = (loss(1e-4) - loss(-1e-4)) / 2e-4
        g, e = got[2 + i].double(), want[2 + i][1]
        assert abs(float((g * d).sum()) - diff) <= float((e * d.abs()).sum()) + 1e-4 * abs(diff) + 1e-3


@types
def test_masked_infinities(dtype):
    """Earlier tokens do not see later ones, nor those that have left their window;
    infinities there reach neither their rows nor their gradients."""
    for D in (64, 128, 40):
        q, k, v, do, _ = _leaves(dtype, B=1, S=150, D=D)
        plain = _run(q, k, v, do, None, window=40, first=2)
        k2, v2 = k.clone(), v.clone()
        for t in (k2, v2):
            t[:, 100] = math.inf
            t[:, 100, :, ::2] = math.nan
        got = _run(q, k2, v2, do, None, window=40, first=2)
        for i in (0, 1, 2):  # out, lse, dq
            assert torch.equal(got[i][:, :100], plain[i][:, :100]) and torch.equal(got[i][:, 140:], plain[i][:, 140:])
        assert bool(torch.isnan(got[0][:, 100:140]).all())


@types
def test_strides_and_shared_rows(dtype):
    """q, k, v as views of one projection; gradients come back in its shape."""
    g = torch.Generator(device=DEV).manual_seed(3)
    for D, pad in ((64, 0), (128, 4), (40, 1)):
        x = torch.randn(2, 60, 4 + 2 + 2, D + pad, generator=g, device=DEV).to(dtype).requires_grad_(True)
        q, k, v = x[:, :, :4, :D], x[:, :, 4:6, :D], x[:, :, 6:, :D]
        do = torch.randn(60, 2, 4, D, generator=g, device=DEV).to(dtype).transpose(0, 1)
        out, lse = ops_amd.window_attention(q, k, v, window=25)
        dx = torch.autograd.grad(out, x, do)[0]
        got = [out.detach(), lse.detach(), dx[:, :, :4, :D], dx[:, :, 4:6, :D], dx[:, :, 6:, :D]]
        ref.check_all(got, ref.window(q.detach(), k.detach(), v.detach(), do, None, 25, 0, None, None, None, dtype,
                                      2.0 ** -8 if dtype == BF else 0.0))


@types
def test_broadcast_inputs(dtype):
    """k and v expanded over the batch: the gradient of the one row is the sum."""
    q, k, v, do, _ = _leaves(dtype, B=3, S=50, D=64)
    k1, v1 = k[:1].clone().requires_grad_(True), v[:1].clone().requires_grad_(True)
    out, _ = ops_amd.window_attention(q, k1.expand_as(k), v1.expand_as(v))
    got = torch.autograd.grad(out, [k1, v1], do)
    want = ref.window(q, k1.detach().expand_as(k), v1.detach().expand_as(v), do, None, dtype=dtype, w=2.0 ** -8 if dtype == BF else 0.0)
    for x, (y, e) in zip(got, want[3:5]):
        h = ref.half(dtype)  # the three gradients' sum rounds once or twice more
        err = (x.double() - y.sum(0, keepdim=True)).abs() - (e.sum(0, keepdim=True) * (1 + 2 * h) + 2 * h * y.abs().sum(0, keepdim=True))
        assert float(err.max()) <= 0.0


def test_equal_calls_give_equal_bits():
    for D, S in ((128, 700), (64, 300)):
        x = _leaves(BF, S=S, D=D, Hq=8)
        a, b = _run(*x, window=200, first=4), _run(*x, window=200, first=4)
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_empty_batches():
    q, k, v, do, sink = _leaves(BF, S=8)
    for cut in (lambda t: t[:0], lambda t: t[:, :0]):
        got = _run(cut(q), cut(k), cut(v), cut(do), sink)
        assert got[2].shape == cut(q).shape and float(got[5].abs().sum()) == 0.0


def test_no_gradient_wanted():
    q, k, v, do, sink = _leaves(BF)
    out, lse = ops_amd.window_attention(q, k, v, attn_sink=sink)
    assert not out.requires_grad
    out, _ = ops_amd.window_attention(q, k, v.requires_grad_(True), attn_sink=sink)
    out.backward(do)
    assert v.grad is not None and q.grad is None
