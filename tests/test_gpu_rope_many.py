"""GPU tests of the rotation and the norms on calls of more row groups than waves
that stay on the card, where several are in flight per wave; tolerances as
derived in test_gpu_rope.py."""
import pytest
import torch

import ops_amd
from tests.test_gpu_rope import BF16, DEV, F32, _bwd_ref, _close, _fwd_ref, _g, _half, _inputs, _randn

pytestmark = pytest.mark.gpu

CASES = [
    # B, S, Hq, Hkv, D, R, off, interleaved, q norm, k norm, dtype, weight dtype
    (2, 2100, 12, 3, 64, 64, 0, True, 64, 64, BF16, BF16),
    (1, 3001, 9, 2, 128, 128, 0, False, 128, 128, BF16, F32),
    (1, 2500, 5, 1, 64, 32, 0, False, 64, 64, F32, F32),
    (1, 2500, 7, 1, 192, 64, 128, False, 192, 128, BF16, BF16),
    (1, 1201, 33, 2, 576, 64, 512, True, 0, 512, BF16, BF16),
    (1, 5000, 3, 1, 64, 64, 0, True, 0, 64, BF16, BF16),  # a side without a norm
    (3, 1777, 8, 1, 64, 64, 0, True, 0, 0, BF16, BF16),
    (1, 4099, 1, 1, 512, 512, 0, True, 512, 0, BF16, BF16),
    (1, 4099, 1, 2, 32, 16, 16, False, 16, 32, F32, F32),
]


@pytest.mark.parametrize("c", CASES, ids=[f"D{c[4]}R{c[5]}{'i' if c[7] else 'h'}n{c[8]}-{c[9]}{str(c[10])[6:]}" for c in CASES])
def test_many_row_groups(c):
    off, inter, dt, wt = c[6], c[7], c[10], c[11]
    q, k, wq, wk, pos, freq = _inputs(c, seed=31)
    leaves = [t if t is None else t.requires_grad_(True) for t in (q, k, wq, wk)]
    yq, yk = ops_amd.qk_norm_rope(q, k, pos, freq, wq, wk, eps=1e-5, rope_offset=off, interleaved=inter)
    g = _g(32)
    dq, dk = _randn(g, *q.shape, dtype=dt), _randn(g, *k.shape, dtype=dt)
    grads = torch.autograd.grad([yq, yk], [t for t in leaves if t is not None], [dq, dk])
    torch.cuda.synchronize()
    dws = list(grads[2:])
    for name, x, w, y, dy, dx in (("q", q, wq, yq, dq, grads[0]), ("k", k, wk, yk, dk, grads[1])):
        x, w = x.detach(), None if w is None else w.detach()
        want, mag, _, _ = _fwd_ref(x, w, pos, freq, 1e-5, off, inter, 1.0)
        _close(y.detach(), want, _half(dt) * want.abs() + 2.0 ** -20 * mag, name)
        wdx, mag, wdw, wmag = _bwd_ref(dy, x, w, pos, freq, 1e-5, off, inter, 1.0)
        _close(dx, wdx, _half(dt) * wdx.abs() + 2.0 ** -18 * mag, "d" + name)
        if w is not None:
            dw, n = dws.pop(0), x[..., 0].numel()
            _close(dw, wdw, _half(wt) * wdw.abs() + (2.0 ** -19 + (n / 1024 + 40) * 2.0 ** -24) * wmag, "dw" + name)


@pytest.mark.parametrize("D,Dv,Hq,Hkv,off,R,nk,inter,dt", [
    (128, 128, 9, 2, 0, 128, 128, False, BF16), (576, 0, 16, 1, 512, 64, 512, True, BF16),
    (64, 192, 5, 3, 0, 64, 64, True, BF16), (64, 32, 4, 4, 0, 32, 0, False, F32)])
def test_append_of_many_tokens(D, Dv, Hq, Hkv, off, R, nk, inter, dt):
    """As qk_norm_rope's rows, bit for bit, with q turned in place; every seventh
    token is padding; nothing else in the pool changes."""
    g = _g(33)
    B, S, ps = 2, 2300, 64
    q, k = _randn(g, B, S, Hq, D, dtype=dt), _randn(g, B, S, Hkv, D, dtype=dt)
    v = _randn(g, B, S, Hkv, Dv, dtype=dt) if Dv else None
    wk = (1 + 0.2 * _randn(g, nk)).to(dt) if nk else None
    n = 40
    kc = _randn(g, B * n, ps, Hkv, D, dtype=dt)
    vc = _randn(g, B * n, ps, Hkv, Dv, dtype=dt) if Dv else None
    bt = torch.randperm(B * n, generator=g, device=DEV).view(B, n).to(torch.int32)
    slots = torch.arange(S, device=DEV).flip(0).expand(B, S) + 70
    slots = torch.where(torch.arange(S, device=DEV) % 7 == 3, -1, slots)
    pos, freq = torch.arange(S, device=DEV), ops_amd.rope_frequencies(R, device=DEV)
    kc0, vc0 = kc.clone(), None if vc is None else vc.clone()
    wq, wkk = ops_amd.qk_norm_rope(q, k, pos, freq, None, wk, rope_offset=off, interleaved=inter)
    out = ops_amd.qk_norm_rope_append(q, k, v, kc, vc, bt, slots, pos, freq, None, wk, rope_offset=off, interleaved=inter,
                                      out=q)
    torch.cuda.synchronize()
    assert out is q and torch.equal(out, wq)
    for b in range(B):
        s = (slots[b] >= 0).nonzero()[:, 0]
        e = slots[b][s]
        kc0[bt[b, e // ps].long(), e % ps] = wkk[b, s]
        if vc is not None:
            vc0[bt[b, e // ps].long(), e % ps] = v[b, s]
    assert torch.equal(kc, kc0) and (vc is None or torch.equal(vc, vc0))
