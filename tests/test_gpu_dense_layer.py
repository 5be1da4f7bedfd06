"""A layer's training step on the operators it is made of: qk_norm_rope and window_attention,
forward and backward, against float64; eager, and captured as one graph."""
import math

import pytest
import torch

import ops_amd
from tests import dense_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(D, S, dtype, seed=5):
    B, Hq, Hkv = 2, 8, 2
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, k, v = (torch.randn(B, S, h, D, generator=g, device=DEV).to(dtype) for h in (Hq, Hkv, Hkv))
    wq, wk = (1.0 + 0.1 * torch.randn(D, generator=g, device=DEV) for _ in range(2))
    do = torch.randn(B, S, Hq, D, generator=g, device=DEV).to(dtype)
    sink = torch.randn(Hq, generator=g, device=DEV)
    return [q, k, v, wq.to(dtype), wk.to(dtype), sink], do


def _layer(xs, do, pos, freq, window, lens):
    q, k = ops_amd.qk_norm_rope(xs[0], xs[1], pos, freq, xs[3], xs[4])
    o, lse = ops_amd.window_attention(q, k, xs[2], window=window, first=2, lens=lens, attn_sink=xs[5])
    return [o.detach(), lse.detach(), *torch.autograd.grad(o, xs, do)]


def _plain(xs, do, pos, freq, window, lens):
    xs = [x.detach().double().requires_grad_(True) for x in xs]
    S, G = xs[0].shape[1], xs[0].shape[2] // xs[1].shape[2]
    ang = pos.double()[:, None] * freq.double()
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def turned(x, w):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        a, b = y.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    q, k = turned(xs[0], xs[3]), turned(xs[1], xs[4])
    live = torch.arange(S, device=DEV) < lens[:, None]
    mask = ref.seen(torch.arange(S, device=DEV), S, window, 2) & live[:, None, :]
    s = torch.matmul(q.transpose(1, 2), k.repeat_interleave(G, 2).permute(0, 2, 3, 1).contiguous()) / math.sqrt(q.shape[3])
    s = s.masked_fill(~mask[:, None], -math.inf)
    z = torch.logsumexp(torch.cat((s, xs[5][None, :, None, None].expand(s.shape[0], -1, S, 1)), -1), -1, keepdim=True)
    o = torch.matmul(torch.exp(s - z), xs[2].repeat_interleave(G, 2).transpose(1, 2).contiguous()).transpose(1, 2)
    o = torch.where(live[:, :, None, None], o, 0.0)
    lse = z.squeeze(-1).transpose(1, 2).masked_fill(~live[:, :, None], -math.inf)
    return [o.detach(), lse.detach(), *torch.autograd.grad(o, xs, do.double())]


@pytest.mark.parametrize("D,S", [(64, 90), (128, 150), (96, 70)])
def test_float32_step(D, S):
    """Float32 throughout: a few hundred roundings of the largest value of each result."""
    xs, do = _inputs(D, S, torch.float32)
    lens = torch.tensor([S, S - 31], dtype=torch.int32, device=DEV)
    pos, freq = torch.arange(S, device=DEV) + 1000, ops_amd.rope_frequencies(D, device=DEV)
    got = _layer([x.requires_grad_(True) for x in xs], do, pos, freq, 33, lens)
    for x, y in zip(got, _plain(xs, do, pos, freq, 33, lens)):
        assert torch.equal(torch.isinf(x), torch.isinf(y))
        x, y = (t.double().masked_fill(torch.isinf(y), 0.0) for t in (x, y))
        assert float((x - y).abs().max()) <= 400 * 2.0 ** -24 * float(y.abs().max())


def test_captured_step():
    """Each replay, with new values in place, is the eager step to the bit."""
    D, S = 128, 300
    xs, do = _inputs(D, S, torch.bfloat16)
    lens = torch.tensor([S, S - 31], dtype=torch.int32, device=DEV)
    pos, freq = torch.arange(S, device=DEV), ops_amd.rope_frequencies(D, device=DEV)

    def step():
        return _layer([x.detach().requires_grad_(True) for x in xs], do, pos, freq, 100, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for k in range(4):
        if k > 1:
            xs[0].mul_(0.75)
            lens.sub_(9)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.tanh(torch.randn(512, 512, device=DEV) @ torch.randn(512, 512, device=DEV))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want)), k
