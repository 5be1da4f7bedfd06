"""The operators around the attention that are timed, and the ranges they stand for.

``rotary``     rotary positions on part of each head (forward, or forward + backward)
``norm_rope``  per-head norm of q and k with the rotation in the same pass: a training step
``append``     the same for serving: the k and v rows go straight into the pages of the cache
``tree``       attention of a tree of drafted tokens over a paged cache
``fork``       the losing beams' rows freed, the winners forked into them
``compact``    the pages in use moved to the low end of the pool

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


def listed():
    return [
        # One decode step's rotation of the rope part of 128 heads: a strided view of the query rows. Latency.
        dict(name="rotary_decode", path="rotary", dtype="bf16", B=4, S=1, H=128, W=MLA_DQK, D=MLA_ROPE, R=MLA_ROPE,
             interleaved=True, pos0=32768, step=False),
        # The same part of a training step on a long prompt, positions stretched by a factor of 4.
        dict(name="rotary_step", path="rotary", dtype="bf16", B=1, S=8192, H=128, W=MLA_DQK, D=MLA_ROPE, R=MLA_ROPE,
             interleaved=True, pos0=0, step=True, factor=4.0),
        # A training step in float32 on a short sequence, half of each head rotated: a unit test's size.
        dict(name="norm_rope_f32", path="norm_rope", dtype="f32", B=1, S=256, Hq=4, Hkv=1, D=64, R=32, interleaved=False,
             pos0=0),
        # A training step of grouped-query attention: 32 query heads, 2 kv heads.
        dict(name="norm_rope_gqa", path="norm_rope", dtype="bf16", B=2, S=8192, Hq=32, Hkv=2, D=128, R=128,
             interleaved=False, pos0=0),
        # A decode step of 64 sequences on pages.
        dict(name="append_decode", path="append", attn="gqa", B=64, S=1, prefix=1000, Hq=32, Hkv=2, D=128,
             interleaved=False),
        # A chunk of a prompt behind a cached prefix, latent rows, one rank of eight (16 of 128 heads).
        dict(name="append_mla", path="append", attn="mla", B=1, S=2048, prefix=14336, Hq=16, Hkv=1, D=MLA_DQK,
             interleaved=True),
        # Eight drafted tokens of one sequence over a short context: latency.
        dict(name="tree_small", path="tree", dtype="bf16", attn="gqa", B=1, T=8, lo=2048, hi=2048, Hq=16, Hkv=1, D=128,
             sink=False),
        # A batch of ragged contexts, 16 drafted tokens each.
        dict(name="tree_gqa", path="tree", dtype="bf16", attn="gqa", B=16, T=16, lo=4096, hi=32768, Hq=32, Hkv=2, D=128,
             sink=False),
        # One long context, the widest tree.
        dict(name="tree_long", path="tree", dtype="bf16", attn="gqa", B=1, T=64, lo=131072, hi=131072, Hq=32, Hkv=8,
             D=128, sink=True),
        # Latent attention, 128 heads on one row: the matrix cores' case.
        dict(name="tree_mla", path="tree", dtype="bf16", attn="mla", B=4, T=8, lo=8192, hi=32768, Hq=128, Hkv=1,
             D=MLA_DQK, sink=False),
        # A beam step: 56 losing beams dropped, 8 winners forked into their rows, two layers of K and V pages.
        dict(name="fork_beams", path="fork", B=64, parents=8, lo=1000, hi=3000, layers=2, Hkv=2, D=128),
        # A cache of latent rows compacted after half of its sequences have gone.
        dict(name="compact_pool", path="compact", B=64, lo=2000, hi=6000, layers=2, Hkv=1, D=MLA_DQK),
    ]


def _size(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm; odd ones as likely as any."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: lengths and batch from the whole range, heads and head dims from those that models have."""
    kind = rng.choice(["rotary", "norm_rope", "norm_rope", "append", "append", "tree", "tree", "tree", "tree_mla", "fork",
                       "compact"])
    if kind == "rotary":
        D = rng.choice([64, 128])
        H = rng.choice([16, 32, 128])
        return dict(path="rotary", dtype=rng.choice(["bf16", "f32"]), B=rng.choice([1, 2, 3]), S=_size(rng, 1, 262144 // (D * H) * 64),
                    H=H, W=rng.choice([D, MLA_DQK]), D=D, R=rng.choice([D, D // 2]), interleaved=rng.choice([True, False]),
                    pos0=rng.choice([0, _size(rng, 1, 1000000)]), step=rng.choice([True, False]),
                    factor=rng.choice([1.0, 4.0, 32.0]))
    if kind == "norm_rope":
        Hkv = rng.choice([1, 2, 4, 8])
        D = rng.choice([64, 128])
        return dict(path="norm_rope", dtype=rng.choice(["bf16", "bf16", "f32"]), B=rng.choice([1, 2]), S=_size(rng, 64, 4096),
                    Hq=Hkv * rng.choice([1, 4, 8]), Hkv=Hkv, D=D, R=rng.choice([D, D // 2]),
                    interleaved=rng.choice([True, False]), pos0=rng.choice([0, _size(rng, 1, 1000000)]))
    if kind == "append":
        attn = rng.choice(["gqa", "mla"])
        B = _size(rng, 1, 64)
        S = rng.choice([1, 1, _size(rng, 2, max(2, 2048 // B))])
        Hkv = 1 if attn == "mla" else rng.choice([1, 2, 4, 8])
        return dict(path="append", attn=attn, B=B, S=S, prefix=_size(rng, 1, 2000), Hkv=Hkv,
                    Hq=rng.choice([16, 32, 128]) if attn == "mla" else Hkv * rng.choice([4, 8, 16]),
                    D=MLA_DQK if attn == "mla" else rng.choice([64, 128]), interleaved=rng.choice([True, False]))
    if kind in ("tree", "tree_mla"):
        mla = kind == "tree_mla"
        Hkv = 1 if mla else rng.choice([1, 2, 4, 8])
        Hq = rng.choice([16, 32, 128]) if mla else Hkv * rng.choice([1, 4, 8, 16])
        f32 = not mla and rng.random() < 0.2
        T, B = _size(rng, 1, 8 if mla else 16 if f32 else 64), _size(rng, 1, 4 if mla or f32 else 16)
        hi = _size(rng, 64, 65536)
        hi = max(64, min(hi, (1 << 29 if mla else 1 << 27 if f32 else 1 << 30) // (B * T * Hq * 16)))
        return dict(path="tree", dtype="f32" if f32 else "bf16", attn="mla" if mla else "gqa", B=B, T=T,
                    lo=max(1, hi // rng.choice([1, 2, 4, 16])), hi=hi, Hq=Hq, Hkv=Hkv,
                    D=MLA_DQK if mla else rng.choice([64, 128]), sink=rng.choice([True, False]))
    lo = _size(rng, 60, 2000)
    mla = rng.choice([True, False])
    c = dict(path=kind, B=_size(rng, 4, 64), lo=lo, hi=lo + _size(rng, 1, 3000), layers=rng.choice([1, 2]),
             Hkv=1 if mla else rng.choice([1, 2]), D=MLA_DQK if mla else 128)
    if kind == "fork":
        c["parents"] = max(1, c["B"] // rng.choice([2, 4, 8]))
    return c


# ---- inputs ----

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _freqs(R, factor=1.0):
    """theta^(-2 i / R) with theta stretched by the context's factor, float64."""
    theta = 10000.0 * factor ** (R / (R - 2)) if factor != 1.0 else 10000.0
    return theta ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)


def _positions(c):
    return (c["pos0"] + torch.arange(c["S"], device=DEV, dtype=torch.int32)).expand(c["B"], c["S"]).contiguous()


def _lens(c):
    """Context lengths evenly over [lo, hi], the longest first."""
    return [c["hi"] - (c["hi"] - c["lo"]) * b // max(1, c["B"] - 1) for b in range(c["B"])]


def _weight(g, n, dtype):
    return (1.0 + 0.1 * torch.randn(n, generator=g, device=DEV)).to(dtype)


def _table(g, pages_of, max_pages, num_pages):
    """A block table whose sequences hold pages_of[b] distinct pages in random order, -1 behind them."""
    bt = torch.full((len(pages_of), max_pages), -1, dtype=torch.int32)
    perm = torch.randperm(num_pages, generator=g, device=DEV).to(torch.int32).cpu()
    at = 0
    for b, n in enumerate(pages_of):
        bt[b, :n] = perm[at:at + n]
        at += n
    return bt.to(DEV)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": case, "path": c["path"]}
    if c["path"] == "rotary":
        dt = DTYPES[c["dtype"]]
        s["x"] = _randn(g, c["B"], c["S"], c["H"], c["W"], dtype=dt)[..., c["W"] - c["D"]:]
        s["dy"] = _randn(g, c["B"], c["S"], c["H"], c["D"], dtype=dt) if c["step"] else None
        s["pos"], s["freq"] = _positions(c), _freqs(c["R"], c.get("factor", 1.0))
        if c["step"]:
            s["x"].requires_grad_(True)
    elif c["path"] == "norm_rope":
        dt = DTYPES[c["dtype"]]
        s["q"] = _randn(g, c["B"], c["S"], c["Hq"], c["D"], dtype=dt).requires_grad_(True)
        s["k"] = _randn(g, c["B"], c["S"], c["Hkv"], c["D"], dtype=dt).requires_grad_(True)
        s["wq"] = _weight(g, c["D"], dt).requires_grad_(True)
        s["wk"] = _weight(g, c["D"], dt).requires_grad_(True)
        s["dq"] = _randn(g, c["B"], c["S"], c["Hq"], c["D"], dtype=dt)
        s["dk"] = _randn(g, c["B"], c["S"], c["Hkv"], c["D"], dtype=dt)
        s["pos"], s["freq"] = _positions(c), _freqs(c["R"])
    elif c["path"] == "append":
        B, S, D, mla = c["B"], c["S"], c["D"], c["attn"] == "mla"
        s["q"] = _randn(g, B, S, c["Hq"], D)
        s["k"] = _randn(g, B, S, c["Hkv"], D)
        s["v"] = None if mla else _randn(g, B, S, c["Hkv"], D)
        # latent rows: the norm is the k row's own, over its first 512 dims; the rotation takes the last 64
        s["wq"] = None if mla else _weight(g, D, torch.bfloat16)
        s["wk"] = _weight(g, MLA_DV if mla else D, torch.bfloat16)
        s["off"], R = (D - MLA_ROPE, MLA_ROPE) if mla else (0, D)
        n = (c["prefix"] + S + PAGE - 1) // PAGE
        s["bt"] = _table(g, [n] * B, n, B * n + 3)
        s["kc"] = torch.zeros((B * n + 3, PAGE, c["Hkv"], D), dtype=torch.bfloat16, device=DEV)
        s["vc"] = None if mla else torch.zeros_like(s["kc"])
        s["slots"] = (c["prefix"] + torch.arange(S, device=DEV, dtype=torch.int32)).expand(B, S).contiguous()
        s["freq"] = _freqs(R)
    elif c["path"] == "tree":
        dt, lens, T = DTYPES[c["dtype"]], _lens(c), c["T"]
        n = (c["hi"] + T + PAGE - 1) // PAGE
        pages = [(x + T + PAGE - 1) // PAGE for x in lens]
        s["L"] = c["hi"] + T
        s["bt"] = _table(g, pages, n, sum(pages))
        s["q"] = 2.0 * _randn(g, c["B"], T, c["Hq"], c["D"], dtype=dt)
        s["kc"] = _randn(g, sum(pages), PAGE, c["Hkv"], c["D"], dtype=dt)
        s["vc"] = s["kc"][..., :MLA_DV] if c["attn"] == "mla" else _randn(g, sum(pages), PAGE, c["Hkv"], c["D"], dtype=dt)
        s["ctx"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        # a random tree: node i hangs under one of the 4 nodes before it; the later sequences have fewer nodes
        up = torch.randint(1, 5, (c["B"], T), generator=g, device=DEV).tolist()
        masks = [[1] * T for _ in lens]
        for b in range(c["B"]):
            for i in range(1, T):
                m = masks[b][max(0, i - up[b][i])] | (1 << i)
                masks[b][i] = m - (1 << 64) if m >= 1 << 63 else m
        s["mask"] = torch.tensor(masks, dtype=torch.int64, device=DEV)
        s["nodes"] = torch.tensor([max(1, T - b % 3) for b in range(c["B"])], dtype=torch.int32, device=DEV)
        s["sink"] = _randn(g, c["Hq"], dtype=torch.float32) if c["sink"] else None
    else:
        lens = _lens(c)
        pages = [(x + PAGE - 1) // PAGE for x in lens]
        n = max(pages)
        num = 2 * sum(pages) + c["B"]
        pool = _randn(g, c["layers"], num, PAGE, c["Hkv"], c["D"])
        s["bt"] = _table(g, pages, n, num)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["pools"] = pool
        if c["path"] == "fork":
            s["pools"] = torch.stack([pool, _randn(g, *pool.shape)], 1).flatten(0, 1)  # K and V of each layer
            P = c["parents"]
            s["children"] = torch.arange(P, c["B"], device=DEV, dtype=torch.int32)
            s["parents"] = torch.randint(0, P, (c["B"] - P,), generator=g, device=DEV, dtype=torch.int32)
        else:
            s["bt"][torch.randperm(c["B"], generator=g, device=DEV)[: c["B"] // 2]] = -1
        s["caches"] = list(s["pools"].unbind(0))
        live = s["bt"][s["bt"] >= 0].long()
        s["refs"] = torch.zeros(num, dtype=torch.int32, device=DEV).index_add_(
            0, live, torch.ones_like(live, dtype=torch.int32))
        s["bt0"], s["refs0"] = s["bt"].clone(), s["refs"].clone()
    return s


# ---- the plain forms: elementary torch operations in float32, rounded once ----

def _cos_sin(pos, freq):
    """cos and sin of pos f, [B, S, 1, R / 2] float32: far positions need the angle in 64 bits."""
    a = pos.double()[:, :, None, None] * freq
    return a.cos().float(), a.sin().float()


def _rotate(x, cs, off, R, interleaved, back=False):
    """x (float32) with its dims [off, off + R) rotated by the angles, or by their negatives."""
    cos, sin = cs
    if back:
        sin = -sin
    p = x[..., off:off + R]
    a, b = (p[..., 0::2], p[..., 1::2]) if interleaved else (p[..., :R // 2], p[..., R // 2:])
    y1, y2 = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((x[..., :off], y, x[..., off + R:]), -1)


def _normed(x, w):
    """The first len(w) dims of x divided by their root mean square and scaled by w; xhat and 1 / rms."""
    n = w.shape[0]
    r = torch.rsqrt((x[..., :n] * x[..., :n]).mean(-1, keepdim=True) + EPS)
    h = x[..., :n] * r
    return torch.cat((h * w, x[..., n:]), -1), h, r


def _plain_norm_rope(x, w, cs, c, dy):
    """y, dx, dw of the norm and the rotation of one tensor's heads."""
    xf, wf, n = x.detach().float(), w.detach().float(), w.shape[0]
    u, h, r = _normed(xf, wf)
    y = _rotate(u, cs, 0, c["R"], c["interleaved"])
    du = _rotate(dy.float(), cs, 0, c["R"], c["interleaved"], back=True)
    g = du * wf
    dx = r * (g - h * (g * h).mean(-1, keepdim=True))
    dw = (du * h).reshape(-1, n).sum(0)
    return y.to(x.dtype), dx.to(x.dtype), dw.to(w.dtype)


def _plain_append(s):
    c, R = s["case"], 2 * s["freq"].shape[0]
    cs = _cos_sin(s["slots"], s["freq"])
    q = s["q"].float()
    q = _normed(q, s["wq"].float())[0] if s["wq"] is not None else q
    q = _rotate(q, cs, s["off"], R, c["interleaved"]).to(s["q"].dtype)
    k = _rotate(_normed(s["k"].float(), s["wk"].float())[0], cs, s["off"], R, c["interleaved"]).to(s["k"].dtype)
    page = torch.gather(s["bt"], 1, (s["slots"] // PAGE).long()).long()
    row = (s["slots"] % PAGE).long()
    s["kc"][page, row] = k
    if s["v"] is not None:
        s["vc"][page, row] = s["v"]
    return [q, s["kc"]] + ([] if s["v"] is None else [s["vc"]])


def _plain_tree(s):
    q, B, T, L = s["q"], s["q"].shape[0], s["q"].shape[1], s["L"]
    Hq, Hkv, Dv = q.shape[2], s["kc"].shape[2], s["vc"].shape[3]
    G = Hq // Hkv
    at = torch.arange(L, device=DEV)
    page = s["bt"][:, at // PAGE].long().clamp(min=0)
    k = s["kc"][page, at % PAGE].float().permute(0, 2, 3, 1).contiguous()  # [B, Hkv, D, L]
    v = s["vc"][page, at % PAGE].float().transpose(1, 2)                   # [B, Hkv, L, Dv]
    qf = q.float().view(B, T, Hkv, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, -1)
    z = torch.matmul(qf, k).view(B, Hkv, T, G, L) * (1.0 / math.sqrt(q.shape[3]))
    node = at - s["ctx"][:, None]                                          # [B, L]
    n, t = s["nodes"][:, None, None], torch.arange(T, device=DEV)[None, :, None]
    bit = (s["mask"][:, :, None] >> node.clamp(0, 63)[:, None, :]) & 1
    ok = ((node[:, None] < 0) | ((bit == 1) & (node[:, None] < n))) & (t < n)  # [B, T, L]
    z = z.masked_fill(~ok[:, None, :, None, :], -math.inf)
    m = z.amax(-1, keepdim=True)
    if s["sink"] is not None:
        m = torch.maximum(m, s["sink"].view(1, Hkv, 1, G, 1))
    p = torch.exp(z - m.masked_fill(m == -math.inf, 0.0))
    l = p.sum(-1, keepdim=True)
    live = (t < n)[:, None, :, None, :]
    if s["sink"] is not None:
        l = l + torch.exp(s["sink"].view(1, Hkv, 1, G, 1) - m)
    o = torch.matmul(p.view(B, Hkv, T * G, L), v).view(B, Hkv, T, G, Dv)
    o = torch.where(live, o / l, 0.0)
    lse = torch.where(live, m + torch.log(l), -math.inf)
    out = o.permute(0, 2, 1, 3, 4).reshape(B, T, Hq, Dv).to(q.dtype)
    return out, lse.squeeze(-1).permute(0, 2, 1, 3).reshape(B, T, Hq)


def _plain_fork(s):
    bt, refs, lens, par, chi = s["bt"], s["refs"], s["lens"], s["parents"].long(), s["children"].long()
    # the losing beams' pages lose a reference
    old = bt[chi]
    refs.sub_(torch.zeros_like(refs).index_add_(0, old.clamp(min=0).flatten().long(), (old >= 0).flatten().int()))
    # whole pages are shared, the last one, filled in part, is copied to the lowest free page
    n, full = lens[par], lens[par] // PAGE
    e = torch.arange(bt.shape[1], device=DEV)
    row = torch.where(e < full[:, None], bt[par], -1)
    refs.index_add_(0, row.clamp(min=0).flatten().long(), (row >= 0).flatten().int())
    part = (n % PAGE) > 0
    free = torch.argsort((refs > 0).int(), stable=True)
    new = free[(torch.cumsum(part.int(), 0) - 1).clamp(min=0)]
    src = torch.gather(bt[par], 1, full.clamp(max=bt.shape[1] - 1)[:, None].long())[:, 0].long()
    bt[chi] = torch.where((e == full[:, None]) & part[:, None], new[:, None].int(), row)
    lens[chi] = n
    refs.index_add_(0, new, part.int())
    live = (torch.arange(PAGE, device=DEV) < (n % PAGE)[:, None])[:, :, None, None]
    dst = torch.where(part, new, free[-1])
    s["pools"][:, dst] = torch.where(live, s["pools"][:, src], s["pools"][:, dst])
    return bt, refs, lens, part.new_ones(part.shape, dtype=torch.int32), *s["caches"]


def _plain_compact(s):
    bt, refs = s["bt"], s["refs"]
    bt.copy_(s["bt0"])
    refs.copy_(s["refs0"])
    used = refs > 0
    count = used.sum()
    ids = torch.arange(refs.shape[0], device=DEV)
    src, dst = ids[used & (ids >= count)], ids[~used & (ids < count)]
    to = ids.to(torch.int32).scatter(0, src, dst.int())
    bt.copy_(torch.where(bt >= 0, to[bt.clamp(min=0).long()], bt))
    refs[dst] = refs[src]
    refs[src] = 0
    s["pools"][:, dst] = s["pools"][:, src]
    return bt, refs, count.int().view(1), *s["caches"]


def _run_plain(s):
    c = s["case"]
    if c["path"] == "rotary":
        cs = _cos_sin(s["pos"], s["freq"])
        y = _rotate(s["x"].detach().float(), cs, 0, c["R"], c["interleaved"]).to(s["x"].dtype)
        if not c["step"]:
            return [y]
        return [y, _rotate(s["dy"].float(), cs, 0, c["R"], c["interleaved"], back=True).to(s["x"].dtype)]
    if c["path"] == "norm_rope":
        cs = _cos_sin(s["pos"], s["freq"])
        q, dq, dwq = _plain_norm_rope(s["q"], s["wq"], cs, c, s["dq"])
        k, dk, dwk = _plain_norm_rope(s["k"], s["wk"], cs, c, s["dk"])
        return [q, k, dq, dk, dwq, dwk]
    if c["path"] == "append":
        return _plain_append(s)
    if c["path"] == "tree":
        return list(_plain_tree(s))
    return list(_plain_fork(s) if c["path"] == "fork" else _plain_compact(s))


# ---- the framework's operators ----

def _run_own(s):
    import ops_amd
    c = s["case"]
    if c["path"] == "rotary":
        y = ops_amd.rotary_embedding(s["x"], s["pos"], s["freq"], interleaved=c["interleaved"])
        if not c["step"]:
            return [y]
        return [y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]]
    if c["path"] == "norm_rope":
        q, k = ops_amd.qk_norm_rope(s["q"], s["k"], s["pos"], s["freq"], s["wq"], s["wk"], eps=EPS,
                                    interleaved=c["interleaved"])
        return [q.detach(), k.detach(),
                *torch.autograd.grad([q, k], [s["q"], s["k"], s["wq"], s["wk"]], [s["dq"], s["dk"]])]
    if c["path"] == "append":
        q = ops_amd.qk_norm_rope_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["bt"], s["slots"], s["slots"],
                                        s["freq"], s["wq"], s["wk"], eps=EPS, rope_offset=s["off"],
                                        interleaved=c["interleaved"])
        return [q, s["kc"]] + ([] if s["v"] is None else [s["vc"]])
    if c["path"] == "tree":
        return list(ops_amd.tree_attention_paged(s["q"], s["kc"], s["vc"], s["bt"], s["ctx"], s["mask"], s["nodes"],
                                                 attn_sink=s["sink"]))
    if c["path"] == "fork":
        ops_amd.cache_free(s["bt"], s["refs"], s["children"])
        ok = ops_amd.cache_fork(s["bt"], s["refs"], s["lens"], s["parents"], s["children"], s["caches"])
        return [s["bt"], s["refs"], s["lens"], ok, *s["caches"]]
    s["bt"].copy_(s["bt0"])
    s["refs"].copy_(s["refs0"])
    used = ops_amd.cache_compact(s["bt"], s["refs"], s["caches"])
    return [s["bt"], s["refs"], used, *s["caches"]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----

def work(case):
    c = case
    if c["path"] == "rotary":
        n = c["B"] * c["S"] * c["H"] * c["D"]
        return {"bytes": (4 if c["step"] else 2) * n * (2 if c["dtype"] == "bf16" else 4),
                "flops": 6 * n * (2 if c["step"] else 1)}
    if c["path"] == "norm_rope":
        n = c["B"] * c["S"] * (c["Hq"] + c["Hkv"]) * c["D"]
        return {"bytes": 5 * n * (2 if c["dtype"] == "bf16" else 4), "flops": 26 * n}
    if c["path"] == "append":
        nk = c["B"] * c["S"] * c["Hkv"] * c["D"]
        nq = c["B"] * c["S"] * c["Hq"] * c["D"]
        return {"bytes": 4 * (nq + nk * (1 if c["attn"] == "mla" else 2)), "flops": 8 * (nq + nk)}
    if c["path"] == "tree":
        e = 2 if c["dtype"] == "bf16" else 4
        Dv = MLA_DV if c["attn"] == "mla" else c["D"]
        keys, rows = sum(_lens(c)) + c["B"] * c["T"], c["B"] * c["T"] * c["Hq"]
        return {"bytes": e * (keys * c["Hkv"] * (c["D"] if c["attn"] == "mla" else 2 * c["D"]) + rows * (c["D"] + Dv)) + 4 * rows,
                "flops": 2 * (c["D"] + Dv) * c["T"] * c["Hq"] * (sum(_lens(c)) + c["B"] * c["T"])}
    lens, row = _lens(c), 2 * c["Hkv"] * c["D"] * c["layers"]
    pages = [(x + PAGE - 1) // PAGE for x in lens]
    if c["path"] == "fork":
        n = c["B"] - c["parents"]  # half a page each, of K and V
        return {"bytes": 2 * 2 * row * n * PAGE // 2 + 8 * c["B"] * max(pages), "flops": 0}
    # half of the pages stay; of a pool over twice as large, about three quarters of those move
    return {"bytes": 2 * row * PAGE * sum(pages) * 3 // 8 + 8 * c["B"] * max(pages), "flops": 0}


# ---- float64 from the definitions ----

def _x_angles(pos, freq):
    return torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos.double()[..., None] * freq)[:, :, None]


def _x_turn(x, z, off, interleaved):
    """The rotated dims as complex numbers times z."""
    R = 2 * z.shape[-1]
    p = x[..., off:off + R]
    p = p.unflatten(-1, (R // 2, 2)) if interleaved else p.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(p.contiguous()) * z)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    out = x.clone()
    out[..., off:off + R] = y
    return out


def _x_norm(x, w):
    n = w.shape[0]
    out = x.clone()
    out[..., :n] = x[..., :n] / torch.sqrt(x[..., :n].square().mean(-1, keepdim=True) + EPS) * w.double()
    return out


def _x_tree(s):
    q, c = s["q"].double(), s["case"]
    G, Dv = c["Hq"] // c["Hkv"], s["vc"].shape[3]
    out = torch.zeros(*q.shape[:3], Dv, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=DEV)
    for b, (ctx, nodes) in enumerate(zip(s["ctx"].tolist(), s["nodes"].tolist())):
        n = ctx + nodes
        pg = s["bt"][b, :(n + PAGE - 1) // PAGE].long()
        seen = torch.ones(nodes, n, dtype=torch.bool, device=DEV)
        for i in range(nodes):
            seen[:, ctx + i] = (s["mask"][b, :nodes] >> i) & 1 == 1
        for h in range(c["Hkv"]):
            k = s["kc"][pg, :, h].reshape(-1, c["D"])[:n].double()
            v = s["vc"][pg, :, h].reshape(-1, Dv)[:n].double()
            for j in range(h * G, h * G + G):
                z = (q[b, :nodes, j] @ k.T) / math.sqrt(c["D"])
                z = torch.where(seen, z, -math.inf)
                if s["sink"] is not None:
                    z = torch.cat((z, s["sink"][j].double().expand(nodes, 1)), 1)
                lse[b, :nodes, j] = torch.logsumexp(z, 1)
                out[b, :nodes, j] = torch.exp(z[:, :n] - lse[b, :nodes, j, None]) @ v
    return [out, lse]


def exact(case, seed):
    c = case
    if c["path"] in ("fork", "compact"):
        return None  # whole numbers and moved rows
    s = prepare(case, seed)
    with torch.enable_grad():
        if c["path"] == "rotary":
            z = _x_angles(s["pos"], s["freq"])
            y = _x_turn(s["x"].detach().double(), z, 0, c["interleaved"])
            return [y, _x_turn(s["dy"].double(), z.conj(), 0, c["interleaved"])] if c["step"] else [y]
        if c["path"] == "norm_rope":
            z = _x_angles(s["pos"], s["freq"])
            leaves = [s[n].detach().double().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
            q = _x_turn(_x_norm(leaves[0], leaves[2]), z, 0, c["interleaved"])
            k = _x_turn(_x_norm(leaves[1], leaves[3]), z, 0, c["interleaved"])
            grads = torch.autograd.grad([q, k], leaves, [s["dq"].double(), s["dk"].double()])
            return [q.detach(), k.detach(), *grads]
    if c["path"] == "append":
        z = _x_angles(s["slots"], s["freq"])
        q = s["q"].double() if s["wq"] is None else _x_norm(s["q"].double(), s["wq"])
        q = _x_turn(q, z, s["off"], c["interleaved"])
        k = _x_turn(_x_norm(s["k"].double(), s["wk"]), z, s["off"], c["interleaved"])
        kc, vc = s["kc"].double(), None if s["v"] is None else s["vc"].double()
        for b in range(c["B"]):
            page, row = s["bt"][b, (s["slots"][b] // PAGE).long()].long(), (s["slots"][b] % PAGE).long()
            kc[page, row] = k[b]
            if vc is not None:
                vc[page, row] = s["v"][b].double()
        return [q, kc] + ([] if vc is None else [vc])
    return _x_tree(s)
