"""GPU test of a whole drafting step as one captured graph: pages for the drafted
rows, their k and v into them, the tree's attention, the accepted path kept and the
rest given back.  Replayed on new inputs with eager work between, every replay
equals the eager step on a copy of the state, bit for bit."""
import pytest
import torch

import ops_amd
from tests.test_gpu_rope import BF16, DEV, _g, _randn
from tests.test_gpu_tree import _masks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mla", [False, True], ids=["gqa", "mla"])
def test_captured_drafting_step(mla):
    g = _g(81)
    B, T, ps, maxp, num = 3, 5, 16, 20, 80
    Hq, Hkv, D, R, off, inter = (16, 1, 576, 64, 512, True) if mla else (8, 2, 128, 128, 0, False)
    wk = (1 + 0.2 * _randn(g, 512 if mla else D)).to(BF16)
    freq = ops_amd.rope_frequencies(R, device=DEV)
    q, k, v = _randn(g, B, T, Hq, D, dtype=BF16), _randn(g, B, T, Hkv, D, dtype=BF16), _randn(g, B, T, Hkv, D, dtype=BF16)
    mask, depth = _masks(B, T, 82), torch.tensor([0, 1, 1, 2, 3], device=DEV)
    path = torch.tensor([[0, 2, 3], [0, 1, -1], [0, -1, -1]], dtype=torch.int32, device=DEV)
    taken = (path >= 0).sum(1).to(torch.int32)
    rows, node = torch.arange(B, device=DEV), torch.arange(T, device=DEV)

    def new_state():
        kc = _randn(_g(83), num, ps, Hkv, D, dtype=BF16)
        st = dict(kc=kc, bt=torch.full((B, maxp), -1, dtype=torch.int32, device=DEV), refs=torch.zeros(num, dtype=torch.int32, device=DEV),
                  lens=torch.zeros(B, dtype=torch.int32, device=DEV))
        if not mla:
            st["vc"] = _randn(_g(84), num, ps, Hkv, D, dtype=BF16)
        start = torch.tensor([30, 16, 47], dtype=torch.int32, device=DEV)
        assert ops_amd.cache_extend(st["bt"], st["refs"], st["lens"], start, ps).tolist() == [1] * B
        st["lens"].copy_(start)
        return st

    def step(st):
        kc, lens = st["kc"], st["lens"]
        vc = kc[..., :512] if mla else st["vc"]
        ok = ops_amd.cache_extend(st["bt"], st["refs"], lens, lens + T, ps)
        y = ops_amd.qk_norm_rope_append(q, k, None if mla else v, kc, None if mla else vc, st["bt"], lens[:, None] + node,
                                        lens[:, None] + depth, freq, None, wk, rope_offset=off, interleaved=inter)
        out, lse = ops_amd.tree_attention_paged(y, kc, vc, st["bt"], lens, mask)
        ops_amd.cache_keep_path([kc] if mla else [kc, vc], st["bt"], lens, path)
        lens += taken
        ops_amd.cache_free(st["bt"], st["refs"], rows, lens, page_size=ps)
        return ok, y, out, lse

    warm, st, plain = new_state(), new_state(), new_state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(st)
    for i in range(4):
        for t, seed in ((q, 90), (k, 100), (v, 110)):
            t.copy_(_randn(_g(seed + i), *t.shape, dtype=BF16))
        want = step(plain)
        graph.replay()
        torch.cuda.synchronize()
        assert want[0].tolist() == [1] * B
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert all(torch.equal(st[n], plain[n]) for n in st)
        assert torch.isfinite(held[2]).all() and torch.isfinite(held[3]).all()
    assert plain["lens"].tolist() == [30 + 4 * 3, 16 + 4 * 2, 47 + 4]
