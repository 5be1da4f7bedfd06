"""Dense attention through a window, e4m3 rows and their pages in float64, for the
tests of their kernels, with the bounds that the kernels' roundings add up to.

Units: u = 2^-24, a float32 rounding; h = eps / 2 of the output's type.  For a row
with n visible keys, products of D terms and mag = max_j scale sum_d |q_d k_jd|:

* a score is off by at most e = (D + 8) u mag (D multiplications and additions, the
  factor to base 2 and the exponent's sum), so a weight by a factor exp(2 e) or so
  (its own score and the maximum or LSE that it is measured from);
* exp2 of a float32 argument a has a relative error of |a| u + 2 u: with the
  maximum at most 8 above it, |a| <= 2 mag / ln 2 + 8: 2^-20 covers mag up to 5, and
  mag's part is in e;
* the sums over n keys add (n + 64) u each, in whatever order;
* weights rounded to bf16 for their product add w = 2^-8.
"""
import math

import torch

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def exponents(x):
    """The exponent byte of each row of x (float64 [..., D]): the smallest e >= 16
    with max |x| <= 448 2^(e - 127); infinities and NaN aside."""
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    e = torch.full(a.shape, 16, dtype=torch.int64, device=x.device)
    for k in range(17, 255):
        e = torch.where(a > 448.0 * 2.0 ** (k - 1 - 127), k, e)
    return e


def e4m3(y):
    """float64 rounded to the nearest e4m3 value (up to 448), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def values(pool, scales):
    """The float64 values that the rows of a pool stand for."""
    x = pool.double()
    if scales is None:
        return x
    e = scales.view(torch.uint8).double()
    return x * torch.exp2(e - 127.0)[..., None]


def quantised(x):
    """(bytes, exponent bytes) of rows x of any type."""
    e = exponents(x.double())
    y = e4m3(x.double() * torch.exp2(127.0 - e.double())[..., None])
    return y.float().to(torch.float8_e4m3fn), e.to(torch.uint8)


def logical(pool, scales, row, n):
    """(values [n, H, D], mapped [n]) of a sequence's first n rows."""
    ps = pool.shape[1]
    at = torch.arange(n, device=pool.device)
    pg = row[at // ps].long()
    ok = (pg >= 0) & (pg < pool.shape[0])
    pg = pg.clamp(0, pool.shape[0] - 1)
    x = values(pool[pg, at % ps], None if scales is None else scales[pg, at % ps])
    return x, ok


def seen(pos, n, window, first):
    """[len(pos), n]: row j <= pos, in the window or among the first."""
    j = torch.arange(n, device=pos.device)[None]
    p = pos[:, None]
    ok = j <= p
    return ok if window is None else ok & ((p - j < window) | (j < first))


def head(q, k, v, ok, scale, sink):
    """One head, float64: out, lse, weights, sum w |v|, max scale sum |q k|."""
    v = torch.where(ok.any(0)[:, None], v, 0.0)
    k = torch.where(ok.any(0)[:, None], k, 0.0)
    z = (q @ k.t() * scale).masked_fill(~ok, -math.inf)
    x = z if sink is None else torch.cat((z, sink.expand(z.shape[0], 1)), 1)
    lse = torch.logsumexp(x, 1) if x.shape[1] else torch.full((z.shape[0],), -math.inf, dtype=z.dtype, device=z.device)
    w = torch.exp(z - lse.masked_fill(lse == -math.inf, 0.0)[:, None])
    mag = ((q.abs() @ k.abs().t() * scale) * ok).amax(1) if z.shape[1] else torch.zeros_like(lse)
    return w @ v, lse, w, w @ v.abs(), mag


def chunk(q, kc, vc, bt, ctx, n, window=None, first=0, sink=None, ks=None, vs=None, scale=None):
    """out, lse, sum w |v|, mag and the number of visible rows of a paged chunk."""
    B, S, Hq, D = q.shape
    Hkv, Dv, cap = kc.shape[2], vc.shape[3], bt.shape[1] * kc.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    dev = q.device
    out, pv = torch.zeros(2, B, S, Hq, Dv, dtype=torch.float64, device=dev)
    lse = torch.full((B, S, Hq), -math.inf, dtype=torch.float64, device=dev)
    mag, num = torch.zeros(2, B, S, Hq, dtype=torch.float64, device=dev)
    for b in range(B):
        c = min(max(int(ctx[b]), 0), cap)
        m = S if n is None else min(max(int(n[b]), 0), S)
        if m == 0:
            continue
        keys = min(c + m, cap)
        k, ok = logical(kc, ks, bt[b], keys)
        v, _ = logical(vc, vs, bt[b], keys)
        mask = seen(c + torch.arange(m, device=dev), keys, window, first) & ok
        for h in range(Hq):
            g = h // (Hq // Hkv)
            s = None if sink is None else sink[h].double()
            out[b, :m, h], lse[b, :m, h], _, pv[b, :m, h], mag[b, :m, h] = head(q[b, :m, h].double(), k[:, g], v[:, g], mask,
                                                                               scale, s)
            num[b, :m, h] = mask.sum(1).double()
    return out, lse, pv, mag, num


def row_error(D, mag, num):
    """The relative error of a row's weights, before any rounding of them."""
    return 2 * (D + 8) * U * mag + (1.25 * num + 64) * U + 2.0 ** -20


def check(got, want, D, dtype, w):
    """got (out, lse) against want within the bounds; w: of the weights' rounding."""
    (out, lse), (o, l, pv, mag, num) = got, want
    assert torch.equal(torch.isfinite(lse), torch.isfinite(l))
    assert torch.equal(lse[~torch.isfinite(l)].double(), l[~torch.isfinite(l)])
    assert torch.isfinite(out).all()
    fin = torch.isfinite(l)
    e = row_error(D, mag, num)
    if fin.any():
        d = ((lse.double() - l).abs() - (e + 2.0 ** -21 * (1 + l.abs())))[fin].max()
        assert float(d) <= 0.0, float(d)
    bound = half(dtype) * o.abs() * (1 + w) + (e[..., None] + w) * pv
    err = (out.double() - o).abs()
    assert float((err - bound).max()) <= 0.0, (float((err - bound).max()), float(err.max()))


def window(q, k, v, do, n, win=None, first=0, sink=None, dlse=None, scale=None, dtype=torch.float32, w=0.0):
    """out, lse, dq, dk, dv, dsink of whole sequences, and bounds of each: a list of
    (value, bound) in that order (lse's and dsink's too).  w: the rounding of weights
    and of ds for their products; o is taken as rounded to dtype in delta."""
    B, S, Hq, D = q.shape
    Hkv, Dv = k.shape[2], v.shape[3]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    f64 = dict(dtype=torch.float64, device=q.device)
    r = {x: torch.zeros(s, **f64) for x, s in (("o", (B, S, Hq, Dv)), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape),
                                               ("ds", (Hq,)))}
    e = {x: torch.zeros_like(t) for x, t in r.items()}
    lse = torch.full((B, S, Hq), -math.inf, **f64)
    el = torch.zeros_like(lse)
    h = half(dtype)
    for b in range(B):
        m = S if n is None else min(max(int(n[b]), 0), S)
        if m == 0:
            continue
        ok = seen(torch.arange(m, device=q.device), m, win, first)
        num = ok.sum(1).double()
        for i in range(Hq):
            g = i // (Hq // Hkv)
            qq, kk, vv, go = q[b, :m, i].double(), k[b, :m, g].double(), v[b, :m, g].double(), do[b, :m, i].double()
            s = None if sink is None else sink[i].double()
            o, l, p, pv, mag = head(qq, kk, vv, ok, scale, s)
            er = row_error(D, mag, num)
            r["o"][b, :m, i], lse[b, :m, i] = o, l
            eo = h * o.abs() * (1 + w) + (er[:, None] + w) * pv
            e["o"][b, :m, i], el[b, :m, i] = eo, er + 2.0 ** -21 * (1 + l.abs())
            dl = torch.zeros_like(l) if dlse is None else dlse[b, :m, i].double()
            delta = (go * o).sum(1) - dl
            ed = (go.abs() * eo).sum(1) + (Dv + 8) * U * ((go * o).abs().sum(1) + dl.abs())
            dp = go @ vv.t()
            edp = (Dv + 8) * U * (go.abs() @ vv.abs().t())
            ds = p * (dp - delta[:, None])
            # a weight of the backward: its score and the forward's LSE
            ew = p * (2 * er[:, None] + 2.0 ** -20 * (1 + l.abs())[:, None])
            eds = ew * (dp - delta[:, None]).abs() + p * (edp + ed[:, None] + 4 * U * (dp.abs() + delta.abs()[:, None]))
            sums = (S * (Hq // Hkv) + 64) * U
            r["dq"][b, :m, i] = ds @ kk * scale
            e["dq"][b, :m, i] = (eds + (w + sums) * ds.abs()) @ kk.abs() * scale
            r["dk"][b, :m, g] += ds.t() @ qq * scale
            e["dk"][b, :m, g] += (eds + (w + sums) * ds.abs()).t() @ qq.abs() * scale
            r["dv"][b, :m, g] += p.t() @ go
            e["dv"][b, :m, g] += (ew + (w + sums) * p).t() @ go.abs()
            if s is not None:
                ps = torch.exp(s - l)
                r["ds"][i] -= (ps * delta).sum()
                e["ds"][i] += (ps * (ed + (2 * er + 2.0 ** -19 * (1 + l.abs() + s.abs()) + B * S * U) * delta.abs())).sum()
    for x in ("dq", "dk", "dv"):
        e[x] = e[x] * (1 + h) + h * r[x].abs()
    return [(r["o"], e["o"]), (lse, el)] + [(r[x], e[x]) for x in ("dq", "dk", "dv")] + ([] if sink is None else [(r["ds"], e["ds"])])


def check_all(got, want):
    for name, x, (y, e) in zip(("out", "lse", "dq", "dk", "dv", "dsink"), got, want):
        x = x.double()
        inf = torch.isinf(y)
        assert torch.equal(x[inf], y[inf]), name
        assert torch.isfinite(x[~inf]).all(), name
        err = ((x - y).abs() - e)[~inf]
        assert err.numel() == 0 or float(err.max()) <= 0.0, (name, float(err.max()), float((x - y)[~inf].abs().max()))


def table(lens, ps, num, seed, extra=0, device="cuda"):
    """A block table of distinct pages in random order, -1 behind them."""
    g = torch.Generator().manual_seed(seed)
    pages = [(n + ps - 1) // ps for n in lens]
    bt = torch.full((len(lens), max(1, max(pages)) + extra), -1, dtype=torch.int32)
    perm = torch.randperm(num, generator=g).int()
    at = 0
    for b, n in enumerate(pages):
        bt[b, :n] = perm[at:at + n]
        at += n
    assert at <= num
    return bt.to(device)
