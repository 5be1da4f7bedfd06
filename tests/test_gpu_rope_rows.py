"""GPU test of the rotation on more rows than one launch has waves for (2^32
threads, a wave a row), which rows of odd sizes take; tolerances as derived in
test_gpu_rope.py."""
import pytest
import torch

import ops_amd
from tests.test_gpu_rope import BF16, DEV, _g, _half

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("append", [False, True])
def test_more_rows_than_waves_of_a_launch(append):
    """262145 tokens x 257 heads of 2 dims.  Appended: the rows of one k head beside them."""
    S, H, D, ps = (1 << 18) + 1, 257, 2, 64
    assert S * H > 1 << 26
    g = _g(41)
    x = torch.randn(1, S, H, D, generator=g, device=DEV).to(BF16)
    pos, freq = torch.arange(S, device=DEV), ops_amd.rope_frequencies(D, device=DEV)
    if append:
        n = S // ps + 1
        k, kc = x[:, :, :1], torch.zeros(n, ps, 1, D, dtype=BF16, device=DEV)
        bt = torch.randperm(n, generator=g, device=DEV)[None].to(torch.int32)
        y = ops_amd.qk_norm_rope_append(x, k, None, kc, None, bt, pos, pos, freq)
        assert torch.equal(kc[bt[0].long()].view(-1, D)[:S], y[0, :, 0])
    else:
        y = ops_amd.rotary_embedding(x, pos, freq)
    torch.cuda.synchronize()
    a = (pos.double()[:, None] * freq)[None]  # [1, S, 1]
    c, s = a.cos().float(), a.sin().float()
    x1, x2 = x[..., 0].float(), x[..., 1].float()
    m = (x1.square() + x2.square()).sqrt()
    for i, want in enumerate((x1 * c - x2 * s, x2 * c + x1 * s)):
        # (the reference's own products and sum in float32: 3 roundings, inside 2^-20)
        bad = (y[..., i].float() - want).abs() - (_half(BF16) * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -19 * m)
        assert float(bad.max()) <= 0.0
