"""The drafted-tree attention in float64, whole rows at once, for contexts that an
element-by-element restatement would take too long on."""
import ctypes
import math

import torch

from ops_amd import _lib
from tests.test_ops_host import _pages, _tree


def exact(q, kc, vc, bt, ctx, mask, nodes, scale, sink=None, weights=lambda p: p):
    """out, lse, sum p |v| and max_s scale sum |q k|; weights(p): what becomes of
    exp(z - max) before the product with v (the sum keeps p)."""
    B, T, Hq, D = q.shape
    ps, Hkv, Dv, dev = kc.shape[1], kc.shape[2], vc.shape[3], q.device
    G, cap = Hq // Hkv, bt.shape[1] * ps
    out, pv = torch.zeros(2, B, T, Hq, Dv, dtype=torch.float64, device=dev)
    lse, mag = torch.full((B, T, Hq), -math.inf, dtype=torch.float64, device=dev), torch.zeros(B, T, Hq, dtype=torch.float64, device=dev)
    for b in range(B):
        c = min(max(int(ctx[b]), 0), cap)
        n = T if nodes is None else min(max(int(nodes[b]), 0), T)
        at = torch.arange(min(c + n, cap), device=dev)
        pg = bt[b, at // ps].long()
        there = (pg >= 0) & (pg < kc.shape[0])
        pg = pg.clamp(0, kc.shape[0] - 1)
        node = (at - c).clamp(0, 63)
        seen = there & ((at < c) | ((mask[b][:, None] >> node) & 1).bool()) & (torch.arange(T, device=dev) < n)[:, None]  # [T, keys]
        seen = seen.repeat_interleave(G, 0)
        for g in range(Hkv):
            k, v = kc[pg, at % ps, g].double(), vc[pg, at % ps, g].double()
            r = q[b, :, g * G:(g + 1) * G].reshape(T * G, D).double()
            z = (r @ k.t() * scale).masked_fill(~seen, -math.inf)
            m = z.amax(1, keepdim=True) if z.shape[1] else torch.full((T * G, 1), -math.inf, dtype=torch.float64, device=dev)
            p = torch.exp(z - m.masked_fill(m == -math.inf, 0.0))
            s = sink.double()[g * G:(g + 1) * G].repeat(T)[:, None] if sink is not None else torch.full_like(m, -math.inf)
            s = s.masked_fill((torch.arange(T, device=dev) >= n).repeat_interleave(G)[:, None], -math.inf)
            top = torch.maximum(m, s)
            total = p.sum(1, keepdim=True) * torch.exp(m - top).nan_to_num(0.0) + torch.exp(s - top).nan_to_num(0.0)
            f = torch.where(total > 0, torch.exp(m - top).nan_to_num(0.0) / total, 0.0)
            hs = slice(g * G, (g + 1) * G)
            out[b, :, hs] = (weights(p) @ v * f).view(T, G, Dv)
            pv[b, :, hs] = (p @ v.abs() * f).view(T, G, Dv)
            lse[b, :, hs] = (top + total.log()).view(T, G)
            if z.shape[1]:
                mag[b, :, hs] = ((r.abs() @ k.abs().t() * scale) * seen).amax(1).view(T, G)
    return out, lse, pv, mag


def check(got, want, D, dtype, w, n):
    """As derived in test_gpu_tree.py, for ranges of n keys: each sum along them adds
    up to n roundings (a lane's own sum of weights n / 4 and the joins); w: of the
    weights' own rounding."""
    (out, lse), (o, l, pv, mag) = got, want
    d = (D + 8) * 2.0 ** -24 * mag
    sums = (n / 4 + 64) * 2.0 ** -24
    assert torch.equal(torch.isfinite(lse), torch.isfinite(l)) and torch.isfinite(out).all()
    fin = torch.isfinite(l)
    assert torch.equal(lse[~fin].double(), l[~fin])
    if fin.any():
        assert float(((lse.double() - l).abs() - (d + sums + 2.0 ** -21 * (1 + l.abs())))[fin].max()) <= 0.0
    b = bound(o, pv, d, dtype, w, n)
    err = (out.double() - o).abs()
    assert float((err - b).max()) <= 0.0, (float((err - b).max()), float(err.max()))


def bound(o, pv, d, dtype, w, n):
    return torch.finfo(dtype).eps / 2 * o.abs() + (2 * d[..., None] + w + (1.25 * n + 64) * 2.0 ** -24 + 2.0 ** -20) * pv


def slots(q, kc, vc, bt):
    """How many key ranges the call may cut its batch into, from the size of the
    workspace that the library asks for (partial results of every range)."""
    B, T, Hq, D = q.shape
    shared = vc.data_ptr() == kc.data_ptr()
    a = _tree(B=B, T=T, Hq=Hq, Hkv=kc.shape[2], Dqk=D, Dv=vc.shape[3], v=0x10000 if shared else 0x20000,
              dtype=_lib.SFA_DTYPE_BF16 if q.dtype == torch.bfloat16 else _lib.SFA_DTYPE_F32)
    for n, t in (("q", q), ("k", kc), ("v", vc)):
        for f, st in zip(("sb", "ss", "sh"), t.stride()):
            setattr(a, f"{n}_{f}", st)
    pg = _pages(max_pages=bt.shape[1], bt_sb=bt.shape[1], page_size=kc.shape[1], num_pages=kc.shape[0])
    size = _lib.load().sfa_tree_fwd_workspace_size(ctypes.byref(a), ctypes.byref(pg))
    return size // (T * Hq * (vc.shape[3] + 1) * 4) if size else B
