"""Infinities and NaN in rows that some tokens see and others do not, in the backward of
dense attention."""
import math

import pytest
import torch

from tests import dense_ref as ref
from tests.test_gpu_window import BF, F32, _leaves, _run

pytestmark = pytest.mark.gpu


def _same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("key", [5, 20, 40, 63, 70, 110, 500, 555])
def test_a_key_that_some_rows_see(D, value, key):
    """Its element is cleared where sums take rows that do not see it, once every wave has made
    its scores of it: tokens that see it get what their score says, each time; the others are
    within their bounds of the values without it.  (Not the same bits: an infinite score moves the
    running maxima of all rows of a wave at once, where a row's own would move later.  What is
    measured from another maximum rounds otherwise, within the same bounds.)"""
    x = _leaves(BF, B=1, S=600, Hq=8, Hkv=2, D=D, sink=False)
    want = ref.window(*x[:4], None, dtype=BF, w=2.0 ** -8)
    k = x[1].clone()
    k[0, key, 0, 3] = value
    y = (x[0], k, *x[2:])
    got = _run(*y)
    for _ in range(4):
        assert all(_same(a, b) for a, b in zip(got, _run(*y)))
    out, lse, dq = got[:3]
    for t, (p, e) in zip((out, lse, dq), want):
        for part in (slice(0, key), slice(None)), (slice(None), slice(4, 8)):
            assert float(((t.double() - p).abs() - e)[:, part[0], part[1]].max()) <= 0.0
    score = x[0][0, key:, :4, 3].double() * value
    gone = score == -math.inf  # (a weight of 0: the token's other rows make its result)
    assert torch.isfinite(dq[0, key:, :4, 4:])[gone].all() and torch.isfinite(out[0, key:, :4])[gone].all()
    assert torch.isnan(dq[0, key:, :4])[~gone].all() and torch.isnan(lse[0, key:, :4])[~gone].all()


@pytest.mark.parametrize("dtype,D,Dv", [(BF, 64, 64), (BF, 128, 128), (BF, 40, 40), (F32, 64, 64), (BF, 192, 160), (F32, 300, 300)])
@pytest.mark.parametrize("which", [1, 2])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_padding_beside_rows_of_infinities(dtype, D, Dv, which, value):
    """A row of k or v that is no number, of a key that every live token of a later row block
    sees: padded tokens of that block keep their zeros."""
    S, lens = 700, torch.tensor([600, 700, 3], dtype=torch.int32, device="cuda")
    x = list(_leaves(dtype, B=3, S=S, Hq=4, Hkv=2, D=D, Dv=Dv))
    x[which] = x[which].clone()
    x[which][:, 1, :, ::3] = value
    out, lse, dq, dk, dv = _run(*x, lens=lens)[:5]
    for t in (out, dq, dk, dv):
        assert not t[0, 600:].any() and not t[2, 3:].any()
    assert bool((lse[0, 600:] == -math.inf).all())
    assert torch.isnan(dq[1, 1:]).any()
