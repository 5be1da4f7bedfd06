"""Gradients of dense attention at row and head counts whose launches would pass 2^32 threads."""
import pytest
import torch

import ops_amd

pytestmark = pytest.mark.gpu


def _r(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").clamp(-6.0, 6.0)


def test_more_than_2_28_rows():
    """A window of one: a token's result is its own v and the gradient of v is do, but for the
    weight, exp of a score and the LSE made of it: up to 36 * 1.4427, four roundings of each
    (2^-24), are 2^-17; dq and dk are differences of two equal numbers of up to 6 * 6, weighed
    with that error, times a row of up to 6."""
    g = torch.Generator(device="cuda").manual_seed(0)
    S, H = 1 << 22, 65
    q, k, v, do = (_r(g, 1, S, H, 1) for _ in range(4))
    xs = [t.requires_grad_(True) for t in (q, k, v)]
    out, lse = ops_amd.window_attention(*xs, window=1)
    dq, dk, dv = torch.autograd.grad(out, xs, do)
    with torch.no_grad():
        assert float((lse - (q * k).squeeze(-1)).abs().max()) <= 2.0 ** -17
        assert float(((out - v).abs() - 2.0 ** -16 * v.abs()).max()) <= 0.0
        assert float(((dv - do).abs() - 2.0 ** -16 * do.abs()).max()) <= 0.0
        assert float(dq.abs().max()) <= 36 * 2.0 ** -16 * 6 and float(dk.abs().max()) <= 36 * 2.0 ** -16 * 6


def test_more_than_2_22_heads():
    """One token a head: its weight beside the sink's, and the sink's gradient -p_sink p do v."""
    g = torch.Generator(device="cuda").manual_seed(1)
    H = (1 << 22) + 37
    q, k, v, do = (_r(g, 1, 1, H, 1) for _ in range(4))
    sink = _r(g, H).requires_grad_(True)
    out, _ = ops_amd.window_attention(q, k, v, attn_sink=sink)
    ds, = torch.autograd.grad(out, sink, do)
    with torch.no_grad():
        z, s = (q * k).double().flatten(), sink.double()
        p = torch.sigmoid(z - s)
        x = (do.double() * v.double()).flatten()
        want = -(1 - p) * p * x
        # (scores up to 36 and a sink of 6, 2^-24 of 42 * 1.4427 for each of some eight roundings: 2^-15.2)
        assert float(((out.flatten().double() - p * v.flatten().double()).abs() - 2.0 ** -15 * p * v.flatten().abs().double()).max()) <= 0.0
        assert float(((ds.double() - want).abs() - 2.0 ** -14 * want.abs() - 2.0 ** -40 * x.abs()).max()) <= 0.0
