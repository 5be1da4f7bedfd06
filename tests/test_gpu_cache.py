"""GPU tests of the cache's pages: every operation against a restatement on
plain lists, whole state compared (tables, counts, lengths, every byte of every
pool), and a run of them together with the attention that reads the pages."""
import math
import random

import pytest
import torch

import ops_amd
from tests import ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _state(seed, B=6, maxp=7, num=40, ps=16, rows=((2, 128, torch.bfloat16), (1, 576, torch.bfloat16)), shared=True):
    """Random sequences over a random pool; some pages shared between two rows."""
    r = random.Random(seed)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    caches = [(torch.randn(num, ps, h, d, generator=g, device=DEV) * 50).to(dt) for h, d, dt in rows]
    ids = r.sample(range(num), num)
    bt, lens, refs = [[-1] * maxp for _ in range(B)], [], [0] * num
    for b in range(B):
        n = r.choice([0, 1, ps - 1, ps, ps + 1, r.randint(0, (maxp - 1) * ps)])
        lens.append(n)
        for e in range((n + ps - 1) // ps):
            pg = bt[b - 1][e] if shared and b > 0 and e < lens[b - 1] // ps and r.random() < 0.3 else -1
            if pg < 0:
                pg = ids.pop()
            bt[b][e] = pg
            refs[pg] += 1
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return t(bt), t(refs), t(lens), caches


def _same(m, bt, refs, lens, caches):
    torch.cuda.synchronize()
    assert bt.tolist() == m.bt
    assert refs.tolist() == m.refs
    if lens is not None:
        assert lens.tolist() == m.lens
    for a, b in zip(caches, m.caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


POOLS = [((2, 128, torch.bfloat16), (1, 576, torch.bfloat16)), ((1, 3, torch.float32),), ((1, 5, torch.uint8),)]


@pytest.mark.parametrize("rows", POOLS, ids=["bf16", "f32-12B", "u8-5B"])
@pytest.mark.parametrize("seed", range(3))
def test_fork(seed, rows):
    bt, refs, lens, caches = _state(seed, B=8, rows=rows)
    ops_amd.cache_free(bt, refs, _i([4, 5, 6, 7]))
    lens[4:] = 0
    m = ref.Pages(bt, refs, lens, caches)
    parents, children = [0, 1, 2, 3, 0], [4, 5, 6, 7, 7]
    ok = ops_amd.cache_fork(bt, refs, lens, _i(parents), _i(children), caches)
    assert ok.tolist() == m.fork(parents, children)
    _same(m, bt, refs, lens, caches)


def test_fork_refuses_pairs_that_make_no_sense():
    bt, refs, lens, caches = _state(5, B=6)
    lens[2:] = 0
    ops_amd.cache_free(bt, refs, _i([2, 3, 4, 5]))
    m = ref.Pages(bt, refs, lens, caches)
    parents, children = [0, 0, 9, 1, -1, 0, 2, 1], [2, 2, 3, 1, 4, 6, 5, -3]
    ok = ops_amd.cache_fork(bt, refs, lens, _i(parents), _i(children), caches)
    assert ok.tolist() == m.fork(parents, children)
    _same(m, bt, refs, lens, caches)


def test_fork_runs_out_of_pages():
    """Four children need a page of their own, two are left: in order."""
    ps, num = 16, 6
    caches = [torch.randn(num, ps, 1, 64, device=DEV)]
    bt = _i([[3, 0, -1], [5, -1, -1]] + [[-1] * 3] * 5)
    refs, lens = _i([1, 0, 0, 1, 7, 1]), _i([20, 16, 0, 0, 0, 0, 0])
    m = ref.Pages(bt, refs, lens, caches)
    parents, children = [0, 0, 1, 0, 0], [2, 3, 4, 5, 6]
    ok = ops_amd.cache_fork(bt, refs, lens, _i(parents), _i(children), caches)
    assert ok.tolist() == m.fork(parents, children) == [1, 1, 1, 0, 0]
    _same(m, bt, refs, lens, caches)


@pytest.mark.parametrize("seed", range(3))
def test_free(seed):
    bt, refs, lens, caches = _state(10 + seed)
    m = ref.Pages(bt, refs, lens, caches)
    rows, keep = [3, 0, 3, -1, 99], [20, 16, 20, 0, 0]
    ops_amd.cache_free(bt, refs, _i(rows), _i(keep), page_size=16)
    m.free(rows, keep)
    _same(m, bt, refs, lens, caches)
    ops_amd.cache_free(bt, refs, torch.arange(6, device=DEV))
    m.free(list(range(6)))
    _same(m, bt, refs, lens, caches)
    assert int(refs.sum()) == 0


@pytest.mark.parametrize("seed", range(4))
def test_extend(seed):
    r = random.Random(seed)
    bt, refs, lens, caches = _state(20 + seed, num=34 if seed else 60)
    m = ref.Pages(bt, refs, lens, caches)
    new = [max(0, x + r.choice([-3, 0, 1, 16, 40])) for x in m.lens]
    new[1], new[4] = 7 * 16 + 1, -5  # past the table; negative
    ok = ops_amd.cache_extend(bt, refs, lens, _i(new), 16)
    assert ok.tolist() == m.extend(new)
    _same(m, bt, refs, lens, caches)


@pytest.mark.parametrize("rows", POOLS, ids=["bf16", "f32-12B", "u8-5B"])
@pytest.mark.parametrize("seed", range(3))
def test_compact(seed, rows):
    bt, refs, lens, caches = _state(30 + seed, rows=rows)
    ops_amd.cache_free(bt, refs, _i([1, 3]))
    m = ref.Pages(bt, refs, None, caches)
    used = ops_amd.cache_compact(bt, refs, caches)
    assert int(used) == m.compact()
    _same(m, bt, refs, None, caches)
    assert int((refs > 0).sum()) == int(used) and bool((refs[int(used):] == 0).all())
    again = [bt.clone(), refs.clone()]
    assert int(ops_amd.cache_compact(bt, refs, caches)) == int(used)
    assert torch.equal(bt, again[0]) and torch.equal(refs, again[1])


def test_compact_empty_and_full():
    c = [torch.randn(5, 4, 2, device=DEV)]
    bt, refs = _i([[-1, -1]]), _i([0] * 5)
    assert int(ops_amd.cache_compact(bt, refs, c)) == 0 and bt.tolist() == [[-1, -1]]
    bt, refs = _i([[4, 2], [0, 1], [3, 4]]), _i([1, 1, 1, 1, 2])
    assert int(ops_amd.cache_compact(bt, refs, c)) == 5 and bt.tolist() == [[4, 2], [0, 1], [3, 4]]


def test_large_pool_scans_in_several_steps():
    """More pages than one step of the scans covers (16384), few of them free."""
    num, ps = 40000, 1
    caches = [torch.arange(num, dtype=torch.float32, device=DEV).view(num, 1, 1).clone()]
    refs = torch.ones(num, dtype=torch.int32, device=DEV)
    free = [5, 16383, 16384, 20000, 39999]
    refs[free] = 0
    bt = _i([[-1] * 8, [-1] * 8])
    lens = _i([0, 0])
    m = ref.Pages(bt, refs, lens, caches)
    ok = ops_amd.cache_extend(bt, refs, lens, _i([3, 2]), ps)
    assert ok.tolist() == m.extend([3, 2]) == [1, 1]
    _same(m, bt, refs, lens, caches)
    refs[:30000:2] = 0
    bt[0, 0], bt[1, 1] = 39999, 31
    refs[31] = 1
    m = ref.Pages(bt, refs, lens, caches)
    assert int(ops_amd.cache_compact(bt, refs, caches)) == m.compact()
    _same(m, bt, refs, lens, caches)


@pytest.mark.parametrize("rows", POOLS, ids=["bf16", "f32-12B", "u8-5B"])
def test_copy_pages(rows):
    _, refs, _, caches = _state(40, rows=rows)
    m = ref.Pages(_i([[0]]), refs, None, caches)
    src, dst = [0, 1, 2, 3, 4, 7, 9, -1, 5, 40], [10, 11, 11, 1, 4, 8, 40, 12, 13, 3]
    ops_amd.cache_copy_pages(caches, _i(src), _i(dst))
    m.copy(src, dst)
    torch.cuda.synchronize()
    for a, b in zip(caches, m.caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_copy_pages_many_pairs_strided_pools_and_more_pools_than_one_launch():
    num, ps = 700, 4
    kv = [torch.randn(num, 2, ps, 8, device=DEV) for _ in range(30)]
    caches = [x[:, i] for x in kv for i in range(2)]
    src, dst = list(range(300)), [i + 300 for i in random.Random(1).sample(range(400), 300)]
    want = [c.clone() for c in caches]
    for c in want:
        c[dst] = c[src]
    ops_amd.cache_copy_pages(caches, _i(src), _i(dst))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


@pytest.mark.parametrize("rows", POOLS, ids=["bf16", "f32-12B", "u8-5B"])
def test_keep_path(rows):
    bt, refs, _, caches = _state(50, B=4, shared=False, rows=rows)
    bt = _i([[1, 2, 3, 4, 5, 6, -1], [7, 8, 9, 10, 11, -1, 13], [14, 15, 16, 17, 18, 19, 20], [21, -1, 22, 23, 24, 25, 40]])
    ctx = [10, 60, -1, 12]
    path = [[0, 2, 3, 9, 20, -1], [5, 4, 3, 2, 1, 0], [1, 2, 3, 4, 5, 6], [0, 1, 8, 40, 100, 2]]
    m = ref.Pages(bt, refs, None, caches)
    ops_amd.cache_keep_path(caches, bt, _i(ctx), torch.tensor(path, device=DEV))
    m.keep_path(ctx, path)
    _same(m, bt, refs, None, caches)


def test_state_on_a_captured_graph():
    """Freeing, forking and extending in one graph; each replay against the lists."""
    bt, refs, lens, caches = _state(60, B=6, num=60)
    rows, parents = _i([3, 4, 5]), _i([0, 1, 2])
    new = _i([0] * 6)

    def step():
        ops_amd.cache_free(bt, refs, rows)
        ok = ops_amd.cache_fork(bt, refs, lens, parents, rows, caches)
        return ok, ops_amd.cache_extend(bt, refs, lens, new, 16)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        new.copy_(lens + 5 + i)
        m = ref.Pages(bt, refs, lens, caches)
        graph.replay()
        torch.cuda.synchronize()
        m.free([3, 4, 5])
        assert held[0].tolist() == m.fork([0, 1, 2], [3, 4, 5])
        assert held[1].tolist() == m.extend(new.tolist())
        _same(m, bt, refs, lens, caches)
        lens.copy_(torch.minimum(new, torch.full_like(new, 100)))


@pytest.mark.parametrize("mla", [False, True], ids=["gqa", "mla"])
def test_speculative_decoding_together(mla):
    """Two rounds of drafting as a serving loop makes them: pages for the drafted
    rows, k and v into them, the tree's attention, the accepted path kept, the
    rest given back, a sequence forked, the pool compacted.  The cache then holds
    what a plain loop over accepted tokens writes, and the attention over it
    equals float64 on that."""
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    B, T, ps, maxp, num = 3, 6, 16, 12, 64
    Hq, Hkv, D, Dv = (16, 1, 576, 512) if mla else (8, 2, 128, 128)
    freq = ops_amd.rope_frequencies(64 if mla else D, device=DEV)
    off = 512 if mla else 0
    opts = dict(rope_offset=off, interleaved=mla)
    wk = torch.ones(512 if mla else D, device=DEV, dtype=torch.bfloat16)

    def rnd(*s):
        return torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)

    kc = rnd(num, ps, Hkv, D)
    vc = kc[..., :Dv] if mla else rnd(num, ps, Hkv, D)
    caches = [kc] if mla else [kc, vc]
    vpool = None if mla else vc
    bt, refs = torch.full((B + 1, maxp), -1, dtype=torch.int32, device=DEV), torch.zeros(num, dtype=torch.int32, device=DEV)
    lens = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    rows_k, rows_v = [[] for _ in range(B + 1)], [[] for _ in range(B + 1)]

    def plain(k, v, pos):
        _, kk = ops_amd.qk_norm_rope(k, k, pos, freq, wk, wk, **opts)
        return kk, (kk[..., :Dv] if mla else v)

    # prompts
    n0 = [37, 16, 5, 0]
    S = max(n0)
    assert ops_amd.cache_extend(bt, refs, lens, _i(n0), ps).tolist() == [1] * (B + 1)
    k, v = rnd(B + 1, S, Hkv, D), None if mla else rnd(B + 1, S, Hkv, D)
    pos = torch.arange(S, device=DEV).expand(B + 1, S)
    slots = torch.where(pos < torch.tensor(n0, device=DEV)[:, None], pos, -1)
    ops_amd.qk_norm_rope_append(None, k, v, kc, vpool, bt, slots, pos, freq, None, wk, **opts)
    kk, vv = plain(k, v, pos)
    for b in range(B + 1):
        rows_k[b] += list(kk[b, :n0[b]])
        rows_v[b] += list(vv[b, :n0[b]])
    lens.copy_(_i(n0))

    par = [-1, 0, 0, 1, 2, 4]  # nodes' parents
    depth = [0, 1, 1, 2, 2, 3]
    masks = []
    for i in range(T):
        masks.append((1 << i) | (masks[par[i]] if par[i] >= 0 else 0))
    mask = torch.tensor([masks] * (B + 1), dtype=torch.int64, device=DEV)
    accepted = [[0, 2, 4, 5], [0, 1], [0, 2], [0]]
    for rnd_i in range(2):
        assert ops_amd.cache_extend(bt, refs, lens, lens + T, ps).tolist() == [1] * (B + 1)
        q, k, v = rnd(B + 1, T, Hq, D), rnd(B + 1, T, Hkv, D), None if mla else rnd(B + 1, T, Hkv, D)
        pos = lens[:, None] + torch.tensor(depth, device=DEV)
        slots = lens[:, None] + torch.arange(T, device=DEV)
        qo = ops_amd.qk_norm_rope_append(q, k, v, kc, vpool, bt, slots, pos, freq, None, wk, **opts)
        out, lse = ops_amd.tree_attention_paged(qo, kc, vc, bt, lens, mask)
        kk, vv = plain(k, v, pos)
        for b in range(B + 1):
            ks, vs = torch.stack(rows_k[b] + list(kk[b])), torch.stack(rows_v[b] + list(vv[b]))
            o, l, pv, mag = ref.tree_rows(qo[b], ks, vs, torch.ones(ks.shape[0], dtype=torch.bool, device=DEV),
                                          len(rows_k[b]), T, masks, 1 / math.sqrt(D), None)
            d = (D + 8) * 2.0 ** -24 * mag
            assert float(((lse[b].double() - l).abs() - d - 2.0 ** -21 * (1 + l.abs())).max()) <= 0.0
            assert float(((out[b].double() - o).abs() - 2.0 ** -8 * o.abs() - (2 * d[..., None] + 2.0 ** -8 + 2.0 ** -20) * pv)
                         .max()) <= 0.0
        # the accepted path moves up, the rest of the drafted rows is given back
        path = torch.full((B + 1, 4), -1, dtype=torch.int32, device=DEV)
        for b, a in enumerate(accepted):
            path[b, :len(a)] = _i(a)
            rows_k[b] += [kk[b, i] for i in a]
            rows_v[b] += [vv[b, i] for i in a]
        ops_amd.cache_keep_path(caches, bt, lens, path)
        lens += _i([len(a) for a in accepted])
        ops_amd.cache_free(bt, refs, torch.arange(B + 1, device=DEV), lens, page_size=ps)
        # the last sequence becomes a fork of the first
        ops_amd.cache_free(bt, refs, _i([B]))
        assert ops_amd.cache_fork(bt, refs, lens, _i([rnd_i]), _i([B]), caches).tolist() == [1]
        rows_k[B], rows_v[B] = list(rows_k[rnd_i]), list(rows_v[rnd_i])
        assert int(ops_amd.cache_compact(bt, refs, caches)) == int((refs > 0).sum())
        for b in range(B + 1):
            at = torch.arange(int(lens[b]), device=DEV)
            assert len(rows_k[b]) == at.numel()
            pg = bt[b, at // ps].long()
            assert torch.equal(kc[pg, at % ps], torch.stack(rows_k[b]))
            assert torch.equal(vc[pg, at % ps], torch.stack(rows_v[b]))
    assert int(refs.sum()) == int((bt >= 0).sum())
