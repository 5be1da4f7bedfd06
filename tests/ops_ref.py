"""Float64 restatements of the operators around the attention (rotation and
norms, drafted trees, cache pages), element by element where it matters, for
the tests of their kernels."""
import math

import torch


def rotate(x, pos, freq, off, interleaved, scale=1.0, back=False):
    """x [B, S, H, D] float64 turned by pos [B, S] * freq [R / 2]."""
    R = 2 * freq.numel()
    a = (pos.double()[..., None] * freq)[:, :, None]
    c, s = a.cos() * scale, a.sin() * scale * (-1.0 if back else 1.0)
    y = x.clone()
    for i in range(R // 2):
        d1, d2 = (off + 2 * i, off + 2 * i + 1) if interleaved else (off + i, off + i + R // 2)
        y[..., d1] = x[..., d1] * c[..., i] - x[..., d2] * s[..., i]
        y[..., d2] = x[..., d2] * c[..., i] + x[..., d1] * s[..., i]
    return y


def norm(x, w, eps):
    """(normed x, xhat, 1 / rms) over the first len(w) dims."""
    if w is None:
        return x, None, None
    n = w.numel()
    r = 1.0 / torch.sqrt(x[..., :n].square().mean(-1, keepdim=True) + eps)
    h = x[..., :n] * r
    y = x.clone()
    y[..., :n] = h * w.double()
    return y, h, r


def tree_rows(q, k_rows, v_rows, mapped, ctx, nodes, mask, scale, sink):
    """One sequence: q [T, Hq, D] against k_rows / v_rows [keys, Hkv, D]; mapped
    [keys] bool; mask: T python ints.  Returns out, lse, the bound's sums
    sum p |v| and max_s scale sum |q k| per row."""
    T, Hq, _ = q.shape
    keys, Hkv, _ = k_rows.shape
    Dv = v_rows.shape[2]
    dev = q.device
    out = torch.zeros(T, Hq, Dv, dtype=torch.float64, device=dev)
    pv = torch.zeros_like(out)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=dev)
    mag = torch.zeros(T, Hq, dtype=torch.float64, device=dev)
    seen = torch.zeros(T, keys, dtype=torch.bool, device=dev)
    for t in range(min(T, nodes)):
        seen[t, :ctx] = True
        for j in range(nodes):
            if ctx + j < keys and (mask[t] >> j) & 1:
                seen[t, ctx + j] = True
    seen &= mapped
    for t in range(min(T, nodes)):
        s = seen[t].nonzero()[:, 0]
        for h in range(Hq):
            g = h // (Hq // Hkv)
            kk, vv = k_rows[s, g].double(), v_rows[s, g].double()
            z = kk @ q[t, h].double() * scale
            if s.numel():
                mag[t, h] = (kk.abs() @ q[t, h].double().abs()).max() * scale
            zz = z if sink is None else torch.cat((z, sink[h].double().view(1)))
            if zz.numel() == 0:
                continue
            lse[t, h] = torch.logsumexp(zz, 0)
            p = torch.exp(z - lse[t, h])
            out[t, h] = p @ vv
            pv[t, h] = p @ vv.abs()
    return out, lse, pv, mag


def tree(q, k_cache, v_cache, bt, ctx, mask, nodes, scale, sink=None):
    """The whole batch: out, lse, sum p |v|, max scale sum |q k|."""
    B, T = q.shape[:2]
    ps = k_cache.shape[1]
    cap = bt.shape[1] * ps
    res = []
    for b in range(B):
        c = min(max(int(ctx[b]), 0), cap)
        n = T if nodes is None else min(max(int(nodes[b]), 0), T)
        keys = min(c + n, cap)
        at = torch.arange(keys, device=q.device)
        pg = bt[b, at // ps].long()
        ok = (pg >= 0) & (pg < k_cache.shape[0])
        pg = pg.clamp(0, k_cache.shape[0] - 1)
        res.append(tree_rows(q[b], k_cache[pg, at % ps], v_cache[pg, at % ps], ok, c, n, [int(x) for x in mask[b].tolist()],
                             scale, sink))
    return tuple(torch.stack(x) for x in zip(*res))


class Pages:
    """The pages' state as plain lists, changed one step at a time."""

    def __init__(self, bt, refs, lens, caches):
        self.bt, self.refs, self.lens = bt.tolist(), refs.tolist(), None if lens is None else lens.tolist()
        self.caches = [c.clone() for c in caches]
        self.ps = caches[0].shape[1] if caches else 1

    def _free(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def _ok(self, pg):
        return 0 <= pg < len(self.refs)

    def _len(self, b):
        return min(max(self.lens[b], 0), len(self.bt[b]) * self.ps)

    def copy(self, src, dst):
        n = len(self.refs)
        real = [0 <= s < n and 0 <= d < n for s, d in zip(src, dst)]
        old = [c.clone() for c in self.caches]
        for i, (s, d) in enumerate(zip(src, dst)):
            later = any(real[j] and dst[j] == d for j in range(i + 1, len(src)))
            read = any(real[j] and src[j] == d for j in range(len(src)) if j != i)
            if real[i] and s != d and not later and not read:
                for c, o in zip(self.caches, old):
                    c[d] = o[s]

    def fork(self, parents, children):
        ok = []
        free = self._free()
        taken = 0
        B = len(self.bt)
        for i, (a, c) in enumerate(zip(parents, children)):
            good = (0 <= a < B and 0 <= c < B and c not in children[:i] and c not in parents)
            if good:
                n = self._len(a)
                full, rest = n // self.ps, n % self.ps
                src = self.bt[a][full] if rest else -1
                row = [p if self._ok(p) else -1 for p in self.bt[a][:full]] + [-1] * (len(self.bt[a]) - full)
                if rest and self._ok(src):
                    taken += 1
                    if taken > len(free):
                        good = False
                    else:
                        new = free[taken - 1]
                        self.refs[new] = 1
                        row[full] = new
                        for cc in self.caches:
                            cc[new, :rest] = cc[src, :rest]
                if good:
                    for p in row[:full]:
                        if p >= 0:
                            self.refs[p] += 1
                    self.bt[c], self.lens[c] = row, n
            ok.append(int(good))
        return ok

    def free(self, rows, keep=None):
        for i, r in enumerate(rows):
            if not 0 <= r < len(self.bt):
                continue
            k = 0 if keep is None else (max(keep[i], 0) + self.ps - 1) // self.ps
            for e in range(k, len(self.bt[r])):
                if self._ok(self.bt[r][e]) and self.refs[self.bt[r][e]] > 0:
                    self.refs[self.bt[r][e]] -= 1
                self.bt[r][e] = -1

    def extend(self, new):
        free, at, ok = self._free(), 0, []
        for b, want in enumerate(new):
            if want > len(self.bt[b]) * self.ps:
                ok.append(0)
                continue
            miss = [e for e in range(self._len(b) // self.ps, (max(want, 0) + self.ps - 1) // self.ps)
                    if not self._ok(self.bt[b][e])]
            good = at + len(miss) <= len(free)
            if good:
                for e, p in zip(miss, free[at:]):
                    self.bt[b][e], self.refs[p] = p, 1
            at += len(miss)
            ok.append(int(good))
        return ok

    def compact(self):
        used = [i for i, r in enumerate(self.refs) if r > 0]
        n = len(used)
        src = [i for i in used if i >= n]
        dst = [i for i in range(n) if self.refs[i] == 0]
        to = dict(zip(src, dst))
        for s, d in to.items():
            self.refs[d], self.refs[s] = self.refs[s], 0
            for c in self.caches:
                c[d] = c[s]
        for row in self.bt:
            for e, p in enumerate(row):
                if self._ok(p) and p >= n:
                    row[e] = to.get(p, -1)
        return n

    def keep_path(self, ctx, path):
        for b, row in enumerate(path):
            if ctx[b] < 0:
                continue
            at = {}
            for i, n in enumerate(row):
                if n < 0:
                    continue
                s, d = self._row(b, ctx[b] + n), self._row(b, ctx[b] + i)
                if s and d:
                    at[d] = [c[s[0], s[1]].clone() for c in self.caches]
            for d, vals in at.items():
                for c, v in zip(self.caches, vals):
                    c[d[0], d[1]] = v

    def _row(self, b, slot):
        e = slot // self.ps
        if not 0 <= e < len(self.bt[b]) or not self._ok(self.bt[b][e]):
            return None
        return self.bt[b][e], slot % self.ps
