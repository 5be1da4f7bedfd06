"""Dense attention over latent rows (576 / 512, V the first dims of K) on the bf16
matrix cores against float64 (tests/dense_ref.py derives the tolerances)."""
import math

import pytest
import torch

import ops_amd
from tests import dense_ref as ref
from tests.test_gpu_dense import BF, DEV, _both, _case, _run, _want

pytestmark = pytest.mark.gpu


def _latent(**kw):
    return _case(BF, D=576, Dv=512, Hkv=1, mla=True, **kw)


@pytest.mark.parametrize("heads", [1, 5, 16, 128])
@pytest.mark.parametrize("S,ctx", [(1, (0,)), (1, (63, 64, 900)), (3, (61, 0, 200)), (65, (1,)), (70, (190, 64))])
def test_lengths_and_heads(heads, S, ctx):
    _both(_latent(S=S, ctx=ctx, Hq=heads, page=64, seed=S + heads))


@pytest.mark.parametrize("page", [1, 16, 64, 256])
@pytest.mark.parametrize("window,first", [(None, 0), (1, 0), (64, 0), (100, 3), (65, 64), (129, 70), (30, 1 << 20)])
def test_windows_and_pages(page, window, first):
    _both(_latent(S=9, ctx=(0, 300, 127), Hq=8, page=page, seed=page), window=window, first=first,
          attn_sink=torch.randn(8, device=DEV))


@pytest.mark.parametrize("page", [16, 64])
def test_padding_and_unmapped_pages(page):
    c = _latent(S=6, ctx=(30, 200, 0, 64), n=[6, 0, 2, 9], Hq=16, page=page, extra=2)
    c["bt"][1, 1] = -1
    c["bt"][3, 0] = 1 << 30
    out, lse = _run(c)
    ref.check((out, lse), _want(c), 576, BF, 2.0 ** -8)
    assert not out[1].any() and not out[2, 2:].any() and torch.isinf(lse[1]).all() and torch.isinf(lse[2, 2:]).all()


@pytest.mark.parametrize("B,S,ctx,heads", [(1, 1, 20000, 16), (2, 4, 5000, 32), (1, 300, 2000, 16)])
def test_ranges_of_keys(B, S, ctx, heads):
    """One sequence's keys on many CUs, joined; the same with each row block whole."""
    _both(_latent(S=S, ctx=(ctx,) * B, Hq=heads, page=64))


@pytest.mark.parametrize("page", [1, 16, 64, 256])
@pytest.mark.parametrize("S,ctx,window,first", [(1, (0, 63, 900), None, 0), (70, (1, 130), None, 0), (9, (300, 127, 64), 100, 3),
                                                (5, (5000,), None, 0), (3, (200, 61), 65, 64)])
def test_rows_of_8_bits(page, S, ctx, window, first):
    _both(_latent(fp8=True, S=S, ctx=ctx, Hq=16, page=page, seed=S), window=window, first=first)


def test_8_bit_rows_of_no_scale_and_padding():
    c = _latent(fp8=True, S=70, ctx=(100, 30), n=[70, 20], Hq=16, page=64)
    want = _run(c)
    j = 130  # token 30's own row
    c["ks"][int(c["bt"][0, j // 64]), j % 64, 0] = 255
    out, lse = _run(c)
    assert torch.equal(out[:, :30], want[0][:, :30]) and torch.equal(out[1], want[0][1]) and torch.equal(lse[1], want[1][1])
    assert torch.isnan(out[0, 30:]).all() and torch.isnan(lse[0, 30:]).all()
    assert not out[1, 20:].any() and torch.isinf(lse[1, 20:]).all()


def test_8_bit_rows_of_another_stride():
    """Rows of 8-byte units only take another way, to the same results."""
    c = _latent(fp8=True, S=4, ctx=(200, 70), Hq=16, page=16)
    want = _run(c)
    num, page = c["k"].shape[:2]
    wide = torch.zeros(num, page, 1, 584, device=DEV, dtype=torch.uint8)
    wide[..., 8:] = c["k"].view(torch.uint8)
    k = wide.view(torch.float8_e4m3fn)[..., 8:]
    c.update(k=k, v=k[..., :512])
    got = _run(c)
    assert float((got[1] - want[1]).abs().max()) < 1e-4
    ref.check(got, _want(c), 576, BF, 2.0 ** -8)


def test_rows_of_another_stride():
    """Latent rows inside wider ones, a pool in another order, q and out of other strides."""
    c = _latent(S=7, ctx=(100, 20), Hq=16, page=16)
    num, page = c["k"].shape[:2]
    wide = torch.full((page, num, 1, 640), math.nan, device=DEV, dtype=BF)
    k = wide.transpose(0, 1)[..., 32:608]
    k.copy_(c["k"])
    q = torch.empty(2, 16, 7, 584, device=DEV, dtype=BF).transpose(1, 2)[..., :576]
    q.copy_(c["q"])
    want = _run(c)
    c.update(q=q, k=k, v=k[..., :512])
    out = torch.empty(2, 16, 7, 520, device=DEV, dtype=BF).transpose(1, 2)[..., :512]
    lse = torch.empty(16, 7, 2, device=DEV).permute(2, 1, 0)
    got = _run(c, out=out, lse=lse)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_values_of_their_own():
    """V that are not K's dims take another way, to the same results."""
    c = _latent(S=4, ctx=(70,), Hq=16, page=64)
    a = _run(c)
    c["v"] = c["v"].clone()
    _both(c)
    b = _run(c)
    assert float((a[1] - b[1]).abs().max()) < 1e-4


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("page", [16, 64])
def test_infinities_in_rows_that_some_see(value, page):
    """A row that only later tokens see: the others are as without it, and so are those whose
    score with it is -inf (its weight is exp(-inf) = 0, its other dims are finite); a score of inf
    or NaN leaves no number."""
    c = _latent(S=70, ctx=(100,), Hq=2, page=page)
    want = _run(c)
    j = 130  # token 30's own row
    at = int(c["bt"][0, j // page]), j % page
    c["k"][at[0], at[1], 0, 3] = value
    out, lse = _run(c)
    assert torch.equal(out[:, :30], want[0][:, :30]) and torch.equal(lse[:, :30], want[1][:, :30])
    score = c["q"][0, 30:, :, 3].double() * value
    gone = score == -math.inf
    assert torch.isfinite(lse[0, 30:])[gone].all() and torch.isnan(lse[0, 30:])[~gone].all()
    assert torch.isnan(out[0, 30:])[~gone].all() and torch.isfinite(out[0, 30:, :, 4:])[gone].all()


def test_equal_calls_give_equal_bits():
    c = _latent(S=40, ctx=(3000, 10), Hq=16, page=64)
    a = _run(c)
    for _ in range(3):
        b = _run(c)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_training_row_of_latent_keys():
    """Whole sequences whose v is a view of k."""
    g = torch.Generator(device=DEV).manual_seed(2)
    k = torch.randn(2, 90, 1, 576, generator=g, device=DEV).to(BF)
    q = torch.randn(2, 90, 4, 576, generator=g, device=DEV).to(BF)
    do = torch.randn(2, 90, 4, 512, generator=g, device=DEV).to(BF)
    lens = torch.tensor([90, 41], dtype=torch.int32, device=DEV)
    ql, kl = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    out, lse = ops_amd.window_attention(ql, kl, kl[..., :512], window=33, first=2, lens=lens)
    dq, dk = torch.autograd.grad(out, (ql, kl), do)
    want = ref.window(q, k, k[..., :512], do, lens, 33, 2, None, None, None, BF, 2.0 ** -8)
    got = [out.detach(), lse.detach(), dq]
    for x, (y, e) in zip(got, want[:3]):
        assert float(((x.double() - y).abs() - e)[torch.isfinite(y)].max()) <= 0.0
    (ky, ke), (vy, ve) = want[3], want[4]
    y, e = ky.clone(), ke.clone()
    # (each of the two is rounded to bf16, then their sum)
    y[..., :512] += vy
    e[..., :512] += ve
    e = e + 2.0 ** -8 * (y.abs() + e)
    assert float(((dk.double() - y).abs() - e).max()) <= 0.0
