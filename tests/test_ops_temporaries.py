"""What a call makes of its arguments (rows with a unit stride, converted indices
and weights) is held until the launch: memory that was given back before could
be another thread's by then.  CPU only."""
import torch

import ops_amd
from tests.host_calls import launches  # noqa: F401

B, S, HQ, HK, D = 2, 3, 4, 2, 64


def _rows(h, d=D, grad=False):
    """[B, S, h, d] with a feature stride other than 1."""
    return torch.randn(B, S, d, h).transpose(2, 3).requires_grad_(grad)


def _i(*x):
    return torch.tensor(x, dtype=torch.int64)


def test_everything_lives_until_the_launch(launches):  # noqa: F811
    pos, freq = torch.arange(S), ops_amd.rope_frequencies(D).float()
    w = torch.ones(D, dtype=torch.bfloat16, requires_grad=True)
    kc, vc = torch.randn(9, 16, HK, D), torch.randn(9, 16, HK, D)
    bt, ctx = _i(0, 1, 2, 3).view(B, 2), _i(3, 4)
    ops_amd.rotary_embedding(_rows(HQ), pos, freq)
    ops_amd.rotary_embedding(_rows(HQ), pos, freq, out=torch.empty(B, S, HQ, D))
    y, z = ops_amd.qk_norm_rope(_rows(HQ, grad=True), _rows(HK, grad=True), pos, freq, w, w)
    torch.autograd.backward([y, z], [_rows(HQ), _rows(HK)])
    with torch.no_grad():
        for q in (_rows(HQ), None):
            ops_amd.qk_norm_rope_append(q, _rows(HK), _rows(HK), kc, vc, bt, pos, pos, freq, w if q is not None else None, w)
        ops_amd.tree_attention_paged(_rows(HQ), kc, vc, bt, ctx, torch.ones(B, S, dtype=torch.int64), ctx,
                                     attn_sink=torch.zeros(HQ, dtype=torch.float64))
    bt, refs, lens = bt.int(), torch.ones(9, dtype=torch.int32), ctx.int()
    ops_amd.cache_copy_pages([kc, vc], _i(0, 1), _i(5, 6))
    ops_amd.cache_fork(bt, refs, lens, _i(0), _i(1), [kc, vc])
    ops_amd.cache_free(bt, refs, _i(0, 1), _i(3, 4), page_size=16)
    ops_amd.cache_extend(bt, refs, lens, _i(9, 9), 16)
    ops_amd.cache_compact(bt, refs, [kc, vc])
    ops_amd.cache_keep_path([kc, vc], bt, ctx, _i(0, 1, 1, 0).view(2, 2))
    assert len(launches) == 13
    assert [(fn, lost) for fn, _, lost in launches if lost] == []
