"""An infinite element of v reaches its dim of the tokens that see it, with its sign, and no
other, wherever in the keys' tiles its row lies."""
import math

import pytest
import torch

import ops_amd
from tests import dense_ref as ref
from tests.test_gpu_dense import BF, DEV, F32, _case, _run, _want
from tests.test_gpu_window import _leaves

pytestmark = pytest.mark.gpu

FORMS = [  # dtype, tokens, heads, kv heads, D, Dv, page
    (BF, 1, 8, 2, 128, 128, 64), (BF, 1, 8, 2, 64, 64, 16), (BF, 6, 8, 2, 128, 128, 16), (BF, 6, 8, 2, 64, 64, 64),
    (BF, 9, 12, 2, 128, 128, 64), (BF, 16, 8, 2, 64, 64, 8), (BF, 40, 8, 2, 128, 128, 64), (BF, 100, 4, 2, 64, 64, 16),
    (F32, 3, 4, 2, 96, 40, 16), (BF, 3, 4, 2, 192, 128, 64)]


@pytest.mark.parametrize("form", FORMS, ids=[f"{f[1] * f[2] // f[3]}rows-{f[4]}-{f[6]}" for f in FORMS])
@pytest.mark.parametrize("ctx", [300, 5000])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_an_infinite_value(form, ctx, value):
    dtype, S, Hq, Hkv, D, Dv, page = form
    c = _case(dtype, S=S, ctx=(ctx, 40), Hq=Hq, Hkv=Hkv, D=D, Dv=Dv, page=page)
    c["q"] *= 0.25  # (no weight comes near 0: scores of a few units)
    want = _want(c)
    for j in (0, 37, 131, 255, ctx - 1):
        at = int(c["bt"][0, j // page]), j % page
        old = c["v"][at[0], at[1], 1, 5].clone()
        c["v"][at[0], at[1], 1, 5] = value
        out, lse = _run(c)
        c["v"][at[0], at[1], 1, 5] = old
        mine = out[0, :, Hq // 2:, 5]
        assert bool((mine == value).all()), j
        mine.copy_(want[0][0, :, Hq // 2:, 5])
        ref.check((out, lse), want, D, dtype, 2.0 ** -8 if dtype == BF else 0.0)


@pytest.mark.parametrize("values", [(math.inf, math.inf), (math.inf, -math.inf), (math.nan, 1.0), (math.inf, math.nan)])
@pytest.mark.parametrize("S,window", [(1, None), (1, 200), (12, None), (60, 100)])
def test_two_of_them(values, S, window):
    """Equal infinities stay one, others leave no number."""
    c = _case(BF, S=S, ctx=(400,), Hq=4, Hkv=1, D=128, page=64)
    c["q"] *= 0.25
    for j, x in zip((330, 390), values):
        c["v"][int(c["bt"][0, j // 64]), j % 64, 0, 77] = x if math.isfinite(x) else 0.5
    want = _want(c, window=window)
    for j, x in zip((330, 390), values):
        c["v"][int(c["bt"][0, j // 64]), j % 64, 0, 77] = x
    out, lse = _run(c, window=window)
    seen = [[s for s in range(S) if window is None or 400 + s - j < window] for j in (330, 390)]
    for s in range(S):
        x = [v for v, ok in zip(values, seen) if s in ok and not math.isfinite(v)]
        got = out[0, s, :, 77]
        total = sum(x)
        assert bool(torch.isnan(got).all() if math.isnan(total) else (got == total).all() if x else torch.isfinite(got).all())
        if x:
            got.copy_(want[0][0, s, :, 77])
    ref.check((out, lse), want, 128, BF, 2.0 ** -8)


@pytest.mark.parametrize("S", [12, 16, 300])
def test_whole_sequences(S):
    q, k, v, _, _ = _leaves(BF, B=1, S=S, Hq=4, Hkv=1, D=128)
    q = q * 0.25
    plain = ops_amd.window_attention(q, k, v)
    v = v.clone()
    v[0, 3, 0, 9] = -math.inf
    out, lse = ops_amd.window_attention(q, k, v)
    assert bool((out[0, 3:, :, 9] == -math.inf).all()) and torch.isfinite(out[0, :3]).all()
    out[0, 3:, :, 9] = plain[0][0, 3:, :, 9]
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
