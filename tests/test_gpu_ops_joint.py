"""GPU tests of the rotation and the norms together with the package's sparse
attention, as a training step and a serving loop run them."""
import math

import pytest
import torch

import ops_amd
from tests.test_gpu_rope import BF16, DEV, F32, _g, _randn

pytestmark = pytest.mark.gpu


def _idx(g, B, S, Hkv, K, keys=None):
    """Distinct keys of 0 .. s (or 0 .. keys - 1), -1 behind them."""
    idx = torch.full((B, S, Hkv, K), -1, dtype=torch.int32, device=DEV)
    for s in range(S):
        n = min(K, s + 1 if keys is None else keys)
        idx[:, s, :, :n] = torch.rand(B, Hkv, s + 1 if keys is None else keys, generator=g, device=DEV).argsort(-1)[..., :n].int()
    return idx


def _plain(q, k, v, wq, wk, pos, freq, idx, scale, eps):
    """Norm, rotation (half layout, all dims) and attention in float64 on the CPU, one query at a time."""
    def turn(x, w):
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
        a = (pos.double()[:, None] * freq)[None, :, None]
        h = x.shape[-1] // 2
        return torch.cat((x[..., :h] * a.cos() - x[..., h:] * a.sin(), x[..., h:] * a.cos() + x[..., :h] * a.sin()), -1)

    q, k = turn(q, wq), turn(k, wk)
    B, S, Hq, _ = q.shape
    G = Hq // k.shape[2]
    rows = []
    for b in range(B):
        for s in range(S):
            for h in range(Hq):
                i = idx[b, s, h // G]
                i = i[i >= 0].long()
                p = torch.softmax(k[b, i, h // G] @ q[b, s, h] * scale, 0)
                rows.append(p @ v[b, i, h // G])
    return torch.stack(rows).view(B, S, Hq, -1)


def test_training_step_against_float64():
    """Gradients of q, k, v and both weights through the norms, the rotation and the
    attention, in float32.  A score is off by d = (64 + 8) 2^-24 12 = 2^-14 at most, a weight
    by 2 d, and so a term of a gradient by 2^-13 or so of the magnitudes that enter it
    (weights, dP and delta); these cancel by less than 8 in the attention and by less than 4
    in the norm's backward: 2^-8 of the largest gradient of a tensor, where a missing
    or doubled term is of its order."""
    g = _g(71)
    B, S, Hq, Hkv, D, K = 2, 21, 4, 2, 64, 8
    q, k, v = _randn(g, B, S, Hq, D), _randn(g, B, S, Hkv, D), _randn(g, B, S, Hkv, D)
    wq, wk = 1 + 0.2 * _randn(g, D), 1 + 0.2 * _randn(g, D)
    dout, idx = _randn(g, B, S, Hq, D), _idx(g, B, S, Hkv, K)
    pos, freq = torch.arange(S, device=DEV) + 100, ops_amd.rope_frequencies(D, device=DEV)
    leaves = [t.requires_grad_(True) for t in (q, k, v, wq, wk)]
    y, z = ops_amd.qk_norm_rope(q, k, pos, freq, wq, wk, eps=1e-5)
    out, _ = ops_amd.sparse_flash_attention(y, z, v, idx, 1 / 8)
    grads = torch.autograd.grad(out, leaves, dout)
    torch.cuda.synchronize()
    ref = [t.detach().cpu().double().requires_grad_(True) for t in leaves]
    want = _plain(*ref, pos.cpu(), freq.cpu(), idx.cpu(), 1 / 8, 1e-5)
    wants = torch.autograd.grad(want, ref, dout.cpu().double())
    for name, a, b in zip(("out", "dq", "dk", "dv", "dwq", "dwk"), (out, *grads), (want, *wants)):
        a, b = a.detach().cpu().double(), b.detach()
        assert float((a - b).abs().max()) <= 2.0 ** -8 * float(b.abs().max()), name


@pytest.mark.parametrize("mla", [False, True], ids=["gqa", "mla"])
def test_training_step_is_its_parts(mla):
    """In bf16 the step's gradients are, bit for bit, those of its parts called one
    after the other (latent rows: v is a view of the turned k, whose gradient
    then holds both)."""
    g = _g(72)
    B, S, K = 1, 70, 32
    Hq, Hkv, D, R, off, inter = (128, 1, 576, 64, 512, True) if mla else (16, 2, 128, 128, 0, False)
    q, k = _randn(g, B, S, Hq, D, dtype=BF16), _randn(g, B, S, Hkv, D, dtype=BF16)
    v = None if mla else _randn(g, B, S, Hkv, D, dtype=BF16)
    wk = (1 + 0.2 * _randn(g, 512 if mla else D)).to(BF16)
    wq = None if mla else (1 + 0.2 * _randn(g, D)).to(BF16)
    leaves = [t.requires_grad_(True) for t in (q, k, v, wq, wk) if t is not None]
    pos, freq, scale = torch.arange(S, device=DEV), ops_amd.rope_frequencies(R, device=DEV), 1 / math.sqrt(D)
    idx, dout = _idx(g, B, S, Hkv, K), _randn(g, B, S, Hq, 512 if mla else D, dtype=BF16)

    def turn():
        return ops_amd.qk_norm_rope(q, k, pos, freq, wq, wk, rope_offset=off, interleaved=inter)

    y, z = turn()
    out, _ = ops_amd.sparse_flash_attention(y, z, z[..., :512] if mla else v, idx, scale)
    grads = torch.autograd.grad(out, leaves, dout)
    y, z = turn()
    with torch.no_grad():
        vv = z[..., :512] if mla else v
        o, l = ops_amd.sfa_forward(y, z, vv, idx, scale)
        dy, dz, dv, _ = ops_amd.sfa_backward(y, z, vv, idx, o, l, dout, scale, merge_kv=mla)
    parts = list(torch.autograd.grad([y, z], [t for t in leaves if t is not v], [dy, dz]))
    if not mla:
        parts.insert(2, dv)
    torch.cuda.synchronize()
    assert torch.equal(out.detach(), o)
    assert all(torch.isfinite(t).all() and torch.equal(t, p) for t, p in zip(grads, parts)) and len(grads) == len(parts)


@pytest.mark.parametrize("dt,mla", [(BF16, False), (BF16, True), (F32, False)], ids=["gqa", "mla", "f32"])
def test_serving_over_the_pages_that_append_writes(dt, mla):
    """A prompt in two chunks (the second padded) and a decode step go through the
    cache; the sparse attention over its pages equals, bit for bit, that over rows
    made without a cache."""
    g = _g(73)
    B, ps, K, num = 2, 16, 24, 24
    Hq, Hkv, D, R, off, inter = (128, 1, 576, 64, 512, True) if mla else (8, 2, 64, 64, 0, False)
    n = 45
    kall = _randn(g, B, n, Hkv, D, dtype=dt)
    vall = None if mla else _randn(g, B, n, Hkv, D, dtype=dt)
    wk = (1 + 0.2 * _randn(g, 512 if mla else D)).to(dt)
    freq, opts = ops_amd.rope_frequencies(R, device=DEV), dict(rope_offset=off, interleaved=inter)
    kc = _randn(g, num, ps, Hkv, D, dtype=dt)
    vc = kc[..., :512] if mla else _randn(g, num, ps, Hkv, D, dtype=dt)
    bt = torch.randperm(num, generator=g, device=DEV)[:B * 4].view(B, 4).to(torch.int32)
    qs = []
    for lo, hi, pad in ((0, 30, 0), (30, 44, 3), (44, 45, 0)):
        S = hi - lo + pad
        at = (torch.arange(S, device=DEV) + lo).clamp(max=hi - 1)
        slots = torch.where(torch.arange(S, device=DEV) < hi - lo, at, -1)
        q = _randn(g, B, S, Hq, D, dtype=dt)
        y = ops_amd.qk_norm_rope_append(q, kall[:, at], None if mla else vall[:, at], kc, None if mla else vc, bt, slots, at, freq,
                                        None, wk, **opts)
        qs.append((y, hi))
    pos = torch.arange(n, device=DEV)
    _, z = ops_amd.qk_norm_rope(kall, kall, pos, freq, None, wk, **opts)
    # (as many rows as the table maps, so that both calls are cut alike; latent rows: one memory
    # for k and v, as in the cache)
    pad = bt.shape[1] * ps - n
    kz = torch.cat((z, z[:, :pad]), 1)
    vz = kz[..., :512] if mla else torch.cat((vall, vall[:, :pad]), 1)
    for y, hi in qs:
        idx = _idx(g, B, y.shape[1], Hkv, K, keys=hi)
        got = ops_amd.sfa_forward_paged(y, kc, vc, bt, idx, 0.1)
        want = ops_amd.sfa_forward(y, kz, vz, idx, 0.1)
        torch.cuda.synchronize()
        assert torch.isfinite(got[0]).all() and all(torch.equal(a, b) for a, b in zip(got, want))
