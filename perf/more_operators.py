"""Dense attention around the sparse one, and the 8-bit cache, that are timed, and
the ranges they stand for.

``chunk``   attention of a chunk of new tokens (or one) over a paged cache, whole
            or through a window with the first tokens visible, bf16, float32 or
            8-bit pages
``window``  a training step (forward and backward) of causal attention through a window
``append``  k and v rows normed, turned, quantised into the pages, and read back
``read``    an 8-bit cache's rows as bf16

``run`` computes a case in plain torch operations, or with ``own`` through
``ops_amd``; ``exact`` evaluates it in float64.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
PAGE = 64
MLA_DQK, MLA_DV, MLA_ROPE = 576, 512, 64  # latent row: K is all of it, V its first 512 dims, the last 64 rotated
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
E4M3_MAX = 448.0


def listed():
    return [
        # One decoded token of one sequence over a short context: latency.
        dict(name="decode_one", path="chunk", dtype="bf16", attn="gqa", cache="same", B=1, S=1, lo=2000, hi=2000, Hq=32, Hkv=8,
             D=128, window=0, first=0, sink=False),
        # A decode step of a ragged batch.
        dict(name="decode_batch", path="chunk", dtype="bf16", attn="gqa", cache="same", B=32, S=1, lo=1000, hi=32768, Hq=32,
             Hkv=8, D=128, window=0, first=0, sink=False),
        # A decode step over long contexts in an 8-bit cache.
        dict(name="decode_fp8", path="chunk", dtype="bf16", attn="gqa", cache="fp8", B=4, S=1, lo=65536, hi=131072, Hq=32, Hkv=8,
             D=128, window=0, first=0, sink=True),
        # A chunk of a prompt behind a cached prefix.
        dict(name="prefill", path="chunk", dtype="bf16", attn="gqa", cache="same", B=1, S=2048, lo=14336, hi=14336, Hq=32, Hkv=8,
             D=128, window=0, first=0, sink=False),
        # Ragged chunks of a sliding-window layer over an 8-bit cache, the first 4 tokens visible.
        dict(name="prefill_window", path="chunk", dtype="bf16", attn="gqa", cache="fp8", B=4, S=1000, lo=1, hi=20000, Hq=64, Hkv=8,
             D=64, window=4096, first=4, sink=False),
        # A chunk over latent rows, one rank of eight (16 of 128 heads).
        dict(name="prefill_mla", path="chunk", dtype="bf16", attn="mla", cache="same", B=1, S=512, lo=14336, hi=14336, Hq=16, Hkv=1,
             D=MLA_DQK, window=0, first=0, sink=False),
        # A training step in float32 on short padded sequences: a unit test's size.
        dict(name="step_f32", path="window", dtype="f32", B=2, S=255, lo=100, Hq=4, Hkv=1, D=64, window=64, first=4, sink=True),
        # A sliding-window layer of grouped-query attention.
        dict(name="step_window", path="window", dtype="bf16", B=1, S=8192, lo=8192, Hq=32, Hkv=8, D=128, window=1024, first=4,
             sink=False),
        # A layer that sees everything, padded batch.
        dict(name="step_causal", path="window", dtype="bf16", B=2, S=4096, lo=3500, Hq=32, Hkv=2, D=128, window=0, first=0,
             sink=False),
        # A decode step of 64 young sequences into an 8-bit cache.
        dict(name="append_decode", path="append", attn="gqa", B=64, S=1, prefix=50, Hq=32, Hkv=8, D=128, interleaved=False),
        # A prompt into an 8-bit cache.
        dict(name="append_prompt", path="append", attn="gqa", B=2, S=4001, prefix=0, Hq=32, Hkv=8, D=128, interleaved=False),
        # The contexts of a batch from the 8-bit cache to bf16.
        dict(name="read_batch", path="read", attn="gqa", B=8, lo=10000, hi=30000, Hkv=8, D=128),
    ]


def _size(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm; odd ones as likely as any."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: lengths and batch from the whole range, heads and head dims from those that models have."""
    kind = rng.choice(["decode", "decode", "decode", "prefill", "prefill", "prefill", "mla", "step", "step", "step", "append",
                       "append", "read"])
    window = rng.choice([0, 0, _size(rng, 16, 8192)])
    first = rng.choice([0, 0, 4, _size(rng, 1, 128)]) if window else 0
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 4, 8, 16])
    D = rng.choice([64, 128])
    if kind in ("decode", "prefill", "mla"):
        c = dict(path="chunk", dtype="bf16", attn="gqa", cache=rng.choice(["same", "same", "fp8"]), window=window, first=first,
                 sink=rng.choice([True, False]))
        if kind == "mla":
            Hkv, Hq, D = 1, rng.choice([16, 32, 128]), MLA_DQK
            c.update(attn="mla", cache="same")
        elif rng.random() < 0.15:
            c.update(dtype="f32", cache="same")
        B = _size(rng, 1, 32 if kind == "decode" else 4)
        S = 1 if kind == "decode" else _size(rng, 2, 2048 if kind == "prefill" else 512)
        # scores of a pass: no more than the largest prefill's; float32 an eighth of it
        most = (1 << 28 if kind == "mla" else 1 << 27 if c["dtype"] == "f32" else 1 << 30) // (B * S * Hq)
        hi = max(1, min(_size(rng, 1, 131072), most))
        c.update(B=B, S=S, hi=hi, lo=max(1, hi // rng.choice([1, 2, 4, 16])), Hq=Hq, Hkv=Hkv, D=D)
        return c
    if kind == "step":
        f32 = rng.random() < 0.25
        B = rng.choice([1, 2, 3])
        most = math.isqrt((1 << 27 if f32 else 1 << 30) // (B * Hq))
        S = _size(rng, 17, max(18, min(8192, most)))
        return dict(path="window", dtype="f32" if f32 else "bf16", B=B, S=S, lo=rng.choice([S, max(1, S // 2)]), Hq=Hq, Hkv=Hkv,
                    D=D, window=window, first=first, sink=rng.choice([True, False]))
    if kind == "append":
        attn = rng.choice(["gqa", "mla"])
        B = _size(rng, 1, 64)
        S = rng.choice([1, 1, _size(rng, 2, max(2, 4096 // B))])
        if attn == "mla":
            Hkv, Hq, D = 1, rng.choice([16, 32, 128]), MLA_DQK
        return dict(path="append", attn=attn, B=B, S=S, prefix=_size(rng, 1, 100), Hq=Hq, Hkv=Hkv, D=D,
                    interleaved=rng.choice([True, False]))
    attn = rng.choice(["gqa", "mla"])
    hi = _size(rng, 16, 20000)
    return dict(path="read", attn=attn, B=_size(rng, 1, 8), lo=max(1, hi // rng.choice([1, 2, 16])), hi=hi,
                Hkv=1 if attn == "mla" else Hkv, D=MLA_DQK if attn == "mla" else D)


# ---- inputs ----

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _lens(c):
    """Lengths evenly over [lo, hi], the longest first."""
    hi = c["hi"] if "hi" in c else c["S"]
    return [hi - (hi - c["lo"]) * b // max(1, c["B"] - 1) for b in range(c["B"])]


def _chunk_lens(c):
    """The chunks are full but for every third sequence's, which is one token short (if it has more)."""
    return [max(1, c["S"] - (b % 3 == 1)) for b in range(c["B"])]


def _table(g, pages_of, num_pages):
    """A block table whose sequences hold pages_of[b] distinct pages in random order, -1 behind them."""
    bt = torch.full((len(pages_of), max(pages_of)), -1, dtype=torch.int32)
    perm = torch.randperm(num_pages, generator=g, device=DEV).to(torch.int32).cpu()
    at = 0
    for b, n in enumerate(pages_of):
        bt[b, :n] = perm[at:at + n]
        at += n
    return bt.to(DEV)


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _fp8_pool(x):
    """(e4m3 values, exponents) of a pool [pages, PAGE, H, D]: each row over the
    smallest power of two 2^(e - 127) that brings it to 448 or less."""
    amax = x.float().abs().amax(-1)
    e = torch.frexp(amax / E4M3_MAX)
    exp = torch.where(e.mantissa == 0.5, e.exponent - 1, e.exponent).clamp(min=-111)
    q = torch.ldexp(x.float(), -exp[..., None]).to(torch.float8_e4m3fn)
    return q, (exp + 127).to(torch.uint8)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c, "path": c["path"]}
    if c["path"] == "chunk":
        dt, lens = DTYPES[c["dtype"]], _lens(c)
        pages = [_pages(n + c["S"]) for n in lens]
        num = sum(pages) + 1
        s["bt"] = _table(g, pages, num)
        s["L"] = max(lens) + c["S"]
        s["q"] = 2.0 * _randn(g, c["B"], c["S"], c["Hq"], c["D"], dtype=dt)
        s["kc"] = _randn(g, num, PAGE, c["Hkv"], c["D"], dtype=dt)
        s["vc"] = s["kc"][..., :MLA_DV] if c["attn"] == "mla" else _randn(g, num, PAGE, c["Hkv"], c["D"], dtype=dt)
        s["ks"] = s["vs"] = None
        if c["cache"] == "fp8":
            s["kc"], s["ks"] = _fp8_pool(s["kc"])
            s["vc"], s["vs"] = _fp8_pool(s["vc"])
        s["ctx"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["n"] = torch.tensor(_chunk_lens(c), dtype=torch.int32, device=DEV)
        s["sink"] = _randn(g, c["Hq"], dtype=torch.float32) if c["sink"] else None
    elif c["path"] == "window":
        dt = DTYPES[c["dtype"]]
        s["q"] = (2.0 * _randn(g, c["B"], c["S"], c["Hq"], c["D"], dtype=dt)).requires_grad_(True)
        s["k"] = _randn(g, c["B"], c["S"], c["Hkv"], c["D"], dtype=dt).requires_grad_(True)
        s["v"] = _randn(g, c["B"], c["S"], c["Hkv"], c["D"], dtype=dt).requires_grad_(True)
        s["do"] = _randn(g, c["B"], c["S"], c["Hq"], c["D"], dtype=dt)
        s["lens"] = torch.tensor(_lens(c), dtype=torch.int32, device=DEV)
        s["sink"] = _randn(g, c["Hq"], dtype=torch.float32).requires_grad_(True) if c["sink"] else None
    elif c["path"] == "append":
        B, S, D, mla = c["B"], c["S"], c["D"], c["attn"] == "mla"
        s["q"] = _randn(g, B, S, c["Hq"], D)
        s["k"] = _randn(g, B, S, c["Hkv"], D)
        s["v"] = None if mla else _randn(g, B, S, c["Hkv"], D)
        s["wq"] = None if mla else (1.0 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(torch.bfloat16)
        s["wk"] = (1.0 + 0.1 * torch.randn(MLA_DV if mla else D, generator=g, device=DEV)).to(torch.bfloat16)
        s["off"], R = (D - MLA_ROPE, MLA_ROPE) if mla else (0, D)
        n = _pages(c["prefix"] + S)
        s["L"] = c["prefix"] + S
        s["bt"] = _table(g, [n] * B, B * n + 3)
        s["kc"], s["ks"] = _fp8_pool(_randn(g, B * n + 3, PAGE, c["Hkv"], D))
        s["vc"], s["vs"] = (None, None) if mla else _fp8_pool(_randn(g, B * n + 3, PAGE, c["Hkv"], D))
        s["slots"] = (c["prefix"] + torch.arange(S, device=DEV, dtype=torch.int32)).expand(B, S).contiguous()
        s["lens"] = torch.full((B,), s["L"], dtype=torch.int32, device=DEV)
        s["freq"] = 10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
    else:
        lens = _lens(c)
        pages = [_pages(n) for n in lens]
        s["L"] = max(lens)
        s["bt"] = _table(g, pages, sum(pages) + 1)
        s["kc"], s["ks"] = _fp8_pool(_randn(g, sum(pages) + 1, PAGE, c["Hkv"], c["D"]))
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return s


# ---- the plain forms: elementary torch operations in float32, rounded once ----

def _value(pool, exps):
    """The float32 values that rows of a pool stand for."""
    x = pool.float()
    return x if exps is None else x * torch.exp2(exps.float() - 127.0)[..., None]


def _rows_of(s, pool, exps):
    """[B, L, H, D] float32: the sequences' rows in order (page 0's behind their pages)."""
    at = torch.arange(s["L"], device=DEV)
    page = s["bt"][:, at // PAGE].long().clamp(min=0)
    return _value(pool[page, at % PAGE], None if exps is None else exps[page, at % PAGE])


def _seen(pos, n, c, L):
    """[B, S, L]: row j <= pos of a live token, in the window or among the first."""
    at = torch.arange(L, device=DEV)[None, None]
    p = pos[..., None]
    ok = (at <= p) & (torch.arange(pos.shape[1], device=DEV)[None, :, None] < n[:, None, None])
    if c["window"]:
        ok = ok & ((at < c["first"]) | (p - at < c["window"]))
    return ok


def _plain_chunk(s):
    c, q = s["case"], s["q"]
    B, S, Hq, D = q.shape
    Hkv, G, L = c["Hkv"], c["Hq"] // c["Hkv"], s["L"]
    k = _rows_of(s, s["kc"], s["ks"])
    v = k[..., :MLA_DV] if c["attn"] == "mla" else _rows_of(s, s["vc"], s["vs"])
    pos = s["ctx"][:, None] + torch.arange(S, device=DEV, dtype=torch.int32)
    o, lse = _attend(q.float(), k, v, _seen(pos, s["n"], c, L), s["sink"], 1.0 / math.sqrt(D))[:2]
    return [o.to(q.dtype), lse]


def _attend(q, k, v, seen, sink, scale):
    """o [B, S, Hq, Dv], lse [B, S, Hq] and the weights [B, Hkv, S G, L] of float32 rows."""
    B, S, Hq, D = q.shape
    Hkv, L, Dv = k.shape[2], k.shape[1], v.shape[3]
    G = Hq // Hkv
    qf = q.view(B, S, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, S * G, D)
    z = torch.matmul(qf, k.permute(0, 2, 3, 1).contiguous()).view(B, Hkv, S, G, L) * scale
    z = z.masked_fill(~seen[:, None, :, None, :], -math.inf)
    m = z.amax(-1, keepdim=True)
    sk = None if sink is None else sink.view(1, Hkv, 1, G, 1)
    if sk is not None:
        m = torch.maximum(m, sk)
    m0 = m.masked_fill(m == -math.inf, 0.0)
    p = torch.exp(z - m0)
    l = p.sum(-1, keepdim=True)
    if sk is not None:
        l = l + torch.exp(sk - m0)
    live = seen.any(-1)[:, None, :, None, None]
    p = torch.where(live, p / l, 0.0).view(B, Hkv, S * G, L)
    lse = torch.where(live, m0 + torch.log(l), -math.inf).squeeze(-1).permute(0, 2, 1, 3).reshape(B, S, Hq)
    o = torch.matmul(p, v.transpose(1, 2).contiguous())
    return o.view(B, Hkv, S, G, Dv).permute(0, 2, 1, 3, 4).reshape(B, S, Hq, Dv), lse, p


def _heads(x, Hkv):
    """[B, S, Hq, D] as [B, Hkv, S G, D]."""
    B, S, Hq, D = x.shape
    return x.view(B, S, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)


def _plain_window(s):
    c = s["case"]
    B, S, Hq, D, Hkv = c["B"], c["S"], c["Hq"], c["D"], c["Hkv"]
    G, scale, dt = Hq // Hkv, 1.0 / math.sqrt(c["D"]), s["q"].dtype
    q, k, v, do = (s[n].detach().float() for n in ("q", "k", "v", "do"))
    sink = None if s["sink"] is None else s["sink"].detach()
    pos = torch.arange(S, device=DEV, dtype=torch.int32).expand(B, S)
    o, lse, p = _attend(q, k, v, _seen(pos, s["lens"], c, S), sink, scale)
    delta = (do * o).sum(-1)                                  # [B, S, Hq]
    doh = _heads(do, Hkv)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), doh)
    ds = torch.matmul(doh, v.permute(0, 2, 3, 1).contiguous())
    ds = p * (ds - _heads(delta[..., None], Hkv))
    dq = torch.matmul(ds, k.transpose(1, 2).contiguous()) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), _heads(q, Hkv)) * scale
    dq = dq.view(B, Hkv, S, G, D).permute(0, 2, 1, 3, 4).reshape(B, S, Hq, D)
    res = [o.to(dt), lse, dq.to(dt), dk.transpose(1, 2).to(dt), dv.transpose(1, 2).to(dt)]
    if sink is not None:
        res.append(-torch.where(lse == -math.inf, 0.0, torch.exp(sink - lse) * delta).sum((0, 1)))
    return res


def _rotate(x, pos, freq, off, interleaved):
    """x (float32) with its dims [off, off + R) turned; angles of far positions in 64 bits."""
    R = 2 * freq.shape[0]
    a = pos.double()[:, :, None, None] * freq
    cos, sin = a.cos().float(), a.sin().float()
    p = x[..., off:off + R]
    a, b = (p[..., 0::2], p[..., 1::2]) if interleaved else (p[..., :R // 2], p[..., R // 2:])
    y1, y2 = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((x[..., :off], y, x[..., off + R:]), -1)


def _normed(x, w):
    """The first len(w) dims of x divided by their root mean square and scaled by w."""
    n = w.shape[0]
    r = torch.rsqrt((x[..., :n] * x[..., :n]).mean(-1, keepdim=True) + EPS)
    return torch.cat((x[..., :n] * r * w, x[..., n:]), -1)


def _put(pool, exps, page, row, x):
    """float32 rows quantised into a pool."""
    pool.view(torch.uint8)[page, row], exps[page, row] = (t.view(torch.uint8) for t in _fp8_pool(x))


def _plain_append(s):
    c = s["case"]
    q = s["q"].float() if s["wq"] is None else _normed(s["q"].float(), s["wq"].float())
    q = _rotate(q, s["slots"], s["freq"], s["off"], c["interleaved"]).to(s["q"].dtype)
    k = _rotate(_normed(s["k"].float(), s["wk"].float()), s["slots"], s["freq"], s["off"], c["interleaved"])
    page = torch.gather(s["bt"], 1, (s["slots"] // PAGE).long()).long()
    row = (s["slots"] % PAGE).long()
    _put(s["kc"], s["ks"], page, row, k)
    if s["v"] is not None:
        _put(s["vc"], s["vs"], page, row, s["v"].float())
    return [q, _plain_read(s, s["kc"], s["ks"])] + ([] if s["v"] is None else [_plain_read(s, s["vc"], s["vs"])])


def _plain_read(s, pool, exps):
    there = torch.arange(s["L"], device=DEV)[None] < s["lens"][:, None]
    return torch.where(there[..., None, None], _rows_of(s, pool, exps), 0.0).to(torch.bfloat16)


def _run_plain(s):
    if s["path"] == "chunk":
        return _plain_chunk(s)
    if s["path"] == "window":
        return _plain_window(s)
    if s["path"] == "append":
        return _plain_append(s)
    return [_plain_read(s, s["kc"], s["ks"])]


# ---- the framework's operators ----

def _run_own(s):
    import ops_amd
    c = s["case"]
    window = c.get("window") or None
    if s["path"] == "chunk":
        return list(ops_amd.chunk_attention_paged(s["q"], s["kc"], s["vc"], s["bt"], s["ctx"], s["n"], window=window,
                                                  first=c["first"], attn_sink=s["sink"], k_scales=s["ks"], v_scales=s["vs"]))
    if s["path"] == "window":
        o, lse = ops_amd.window_attention(s["q"], s["k"], s["v"], window=window, first=c["first"], lens=s["lens"],
                                          attn_sink=s["sink"])
        leaves = [s[n] for n in ("q", "k", "v", "sink") if s[n] is not None]
        return [o.detach(), lse.detach(), *torch.autograd.grad(o, leaves, s["do"])]
    if s["path"] == "append":
        q = ops_amd.qk_norm_rope_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["bt"], s["slots"], s["slots"], s["freq"],
                                        s["wq"], s["wk"], eps=EPS, rope_offset=s["off"], interleaved=c["interleaved"],
                                        k_scales=s["ks"], v_scales=s["vs"])
        pools = [(s["kc"], s["ks"])] + ([] if s["v"] is None else [(s["vc"], s["vs"])])
        return [q] + [ops_amd.cache_read(p, s["bt"], s["lens"], s["L"], scales=e) for p, e in pools]
    return [ops_amd.cache_read(s["kc"], s["bt"], s["lens"], s["L"], scales=s["ks"])]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----

def _pairs(c):
    """(visible (token, row) pairs, rows that some token sees) of the case's sequences."""
    pairs = rows = 0
    W, F = c["window"] or 1 << 40, c["first"]
    train = c["path"] == "window"
    for ctx, n in zip([0] * c["B"] if train else _lens(c), _lens(c) if train else _chunk_lens(c)):
        for p in range(ctx, ctx + n):
            lo = max(0, p - W + 1)
            pairs += p + 1 - lo + min(F, lo)
        lo = max(0, ctx - W + 1)
        rows += ctx + n - lo + min(F, lo)
    return pairs, rows


def work(case):
    c = case
    if c["path"] == "chunk":
        pairs, rows = _pairs(c)
        e, ce = 2 if c["dtype"] == "bf16" else 4, 1 if c["cache"] == "fp8" else 2 if c["dtype"] == "bf16" else 4
        Dv = MLA_DV if c["attn"] == "mla" else c["D"]
        tok = c["B"] * c["S"] * c["Hq"]
        kv = rows * c["Hkv"] * (c["D"] if c["attn"] == "mla" else 2 * c["D"]) * ce
        return {"bytes": kv + e * tok * (c["D"] + Dv) + 4 * tok, "flops": 2 * (c["D"] + Dv) * c["Hq"] * pairs}
    if c["path"] == "window":
        pairs, _ = _pairs(c)
        e = 2 if c["dtype"] == "bf16" else 4
        n = c["B"] * c["S"] * c["D"]
        # q, k, v, dout in; out, dq, dk, dv out; two products forward, five backward
        return {"bytes": e * n * (4 * c["Hq"] + 4 * c["Hkv"]), "flops": 14 * c["D"] * c["Hq"] * pairs}
    if c["path"] == "append":
        two = 1 if c["attn"] == "mla" else 2
        nq, nk = c["B"] * c["S"] * c["Hq"] * c["D"], c["B"] * c["S"] * c["Hkv"] * c["D"] * two
        old = c["B"] * c["prefix"] * c["Hkv"] * c["D"] * two
        # q in and out, new rows in and out as bytes; all rows read back as bytes and written as bf16
        return {"bytes": 4 * nq + 3 * nk + old + 2 * (nk + old), "flops": 8 * (nq + nk)}
    n = c["Hkv"] * c["D"]
    return {"bytes": sum(_lens(c)) * n + 2 * c["B"] * c["hi"] * n, "flops": 0}


# ---- float64 from the definitions ----

def _x_values(pool, exps):
    x = pool.to(torch.float64)
    return x if exps is None else torch.ldexp(x, exps.to(torch.int32)[..., None] - 127)


def _x_head(q, k, v, pos, c, sink, scale):
    """One head: out, lse, the weights and the mask of float64 rows q at positions pos over rows k, v."""
    at = torch.arange(k.shape[0], device=DEV)
    seen = at <= pos[:, None]
    if c["window"]:
        seen &= (at > (pos - c["window"])[:, None]) | (at < c["first"])
    z = torch.where(seen, (q @ k.T) * scale, -math.inf)
    lse = torch.logsumexp(z if sink is None else torch.cat((z, sink.double().expand(z.shape[0], 1)), 1), 1)
    w = torch.exp(z - lse[:, None])
    return w @ v, lse, w


def _x_chunk(s):
    c, q = s["case"], s["q"].double()
    G, Dv, scale = c["Hq"] // c["Hkv"], s["vc"].shape[3], 1.0 / math.sqrt(c["D"])
    out = torch.zeros(*q.shape[:3], Dv, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=DEV)
    for b, (ctx, n) in enumerate(zip(s["ctx"].tolist(), s["n"].tolist())):
        pg = s["bt"][b, :_pages(ctx + n)].long()
        pos = ctx + torch.arange(n, device=DEV)
        for h in range(c["Hkv"]):
            k = _x_values(s["kc"][pg, :, h], None if s["ks"] is None else s["ks"][pg, :, h]).flatten(0, 1)[:ctx + n]
            v = _x_values(s["vc"][pg, :, h], None if s["vs"] is None else s["vs"][pg, :, h]).flatten(0, 1)[:ctx + n]
            for j in range(h * G, h * G + G):
                out[b, :n, j], lse[b, :n, j], _ = _x_head(q[b, :n, j], k, v, pos, c, None if s["sink"] is None else s["sink"][j],
                                                          scale)
    return [out, lse]


def _x_window(s):
    c = s["case"]
    G, scale = c["Hq"] // c["Hkv"], 1.0 / math.sqrt(c["D"])
    x = {n: s[n].detach().double() for n in ("q", "k", "v", "do")}
    out, dq = torch.zeros_like(x["q"]), torch.zeros_like(x["q"])
    dk, dv = torch.zeros_like(x["k"]), torch.zeros_like(x["k"])
    lse = torch.full(out.shape[:3], -math.inf, dtype=torch.float64, device=DEV)
    dsink = torch.zeros(c["Hq"], dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        pos = torch.arange(n, device=DEV)
        for j in range(c["Hq"]):
            h = j // G
            q, k, v, do = x["q"][b, :n, j], x["k"][b, :n, h], x["v"][b, :n, h], x["do"][b, :n, j]
            sink = None if s["sink"] is None else s["sink"].detach()[j].double()
            out[b, :n, j], l, w = _x_head(q, k, v, pos, c, sink, scale)
            lse[b, :n, j] = l
            g = do @ v.T
            mean = (w * g).sum(1, keepdim=True)
            if sink is not None:
                dsink[j] -= (torch.exp(sink - l) * mean[:, 0]).sum()
            g = w * (g - mean) * scale
            dq[b, :n, j] = g @ k
            dk[b, :n, h] += g.T @ q
            dv[b, :n, h] += w.T @ do
    return [out, lse, dq, dk, dv] + ([] if s["sink"] is None else [dsink])


def _x_quantised(x):
    """The values that 8 bits hold of float64 rows: 3 bits behind the leading one,
    steps no finer than 2^-9 of the row's scale, ties to even."""
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / E4M3_MAX)))
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def _x_append(s):
    c = s["case"]
    z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["slots"].double()[..., None] * s["freq"])[:, :, None]

    def row(x, w):
        x = x.double()
        if w is not None:
            n = w.shape[0]
            x[..., :n] = x[..., :n] / torch.sqrt(x[..., :n].square().mean(-1, keepdim=True) + EPS) * w.double()
        R = 2 * z.shape[-1]
        p = x[..., s["off"]:s["off"] + R]
        p = p.unflatten(-1, (R // 2, 2)) if c["interleaved"] else p.unflatten(-1, (2, R // 2)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(p.contiguous()) * z)
        x[..., s["off"]:s["off"] + R] = y.flatten(-2) if c["interleaved"] else y.transpose(-1, -2).flatten(-2)
        return x

    res = [row(s["q"], s["wq"])]
    for new, pool, exps in ((row(s["k"], s["wk"]), s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        if new is not None:
            old = torch.stack([_x_values(pool[t], exps[t]).flatten(0, 1)[:c["prefix"]] for t in s["bt"].long()])
            res.append(torch.cat((old, _x_quantised(new.double())), 1))
    return res


def exact(case, seed):
    s = prepare(case, seed)
    if s["path"] == "chunk":
        return _x_chunk(s)
    if s["path"] == "window":
        return _x_window(s)
    if s["path"] == "append":
        return _x_append(s)
    out = torch.zeros(case["B"], s["L"], case["Hkv"], case["D"], dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        pg = s["bt"][b, :_pages(n)].long()
        out[b, :n] = _x_values(s["kc"][pg], s["ks"][pg]).flatten(0, 1)[:n]
    return [out]
