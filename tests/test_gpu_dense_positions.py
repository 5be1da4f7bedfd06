"""Dense attention over a table that ends before the tokens' positions: the rows that the
table does not have are not seen, the others by their true distance."""
import pytest
import torch

from tests import dense_ref as ref
from tests.test_gpu_dense import BF, DEV, F32, _case, _run

pytestmark = pytest.mark.gpu

FORMS = {  # dtype, e4m3, tokens, heads, kv heads, D, Dv, latent
    "few": (BF, False, 2, 8, 2, 128, 128, False), "few-e4m3": (BF, True, 3, 8, 2, 64, 64, False),
    "wide": (BF, False, 40, 8, 2, 128, 128, False), "wide-e4m3": (BF, True, 70, 4, 2, 64, 64, False),
    "latent": (BF, False, 3, 16, 1, 576, 512, True), "latent-e4m3": (BF, True, 5, 16, 1, 576, 512, True),
    "held": (F32, False, 5, 4, 2, 96, 40, False), "any": (BF, False, 5, 4, 2, 192, 128, False)}
TOP = (1 << 31) - 1


def _want(c, ctx, window, first, sink):
    """As ref.chunk, but from the tokens' own positions."""
    B, S, Hq, D = c["q"].shape
    Hkv, Dv, cap = c["k"].shape[2], c["v"].shape[3], c["bt"].shape[1] * c["k"].shape[1]
    out, pv = torch.zeros(2, B, S, Hq, Dv, dtype=torch.float64, device=DEV)
    lse, mag, num = torch.zeros(3, B, S, Hq, dtype=torch.float64, device=DEV)
    for b in range(B):
        k, ok = ref.logical(c["k"], c["ks"], c["bt"][b], cap)
        v, _ = ref.logical(c["v"], c["vs"], c["bt"][b], cap)
        mask = ref.seen(ctx[b] + torch.arange(S, device=DEV), cap, window, first) & ok
        for h in range(Hq):
            g = h // (Hq // Hkv)
            out[b, :, h], lse[b, :, h], _, pv[b, :, h], mag[b, :, h] = ref.head(
                c["q"][b, :, h].double(), k[:, g], v[:, g], mask, D ** -0.5, None if sink is None else sink[h].double())
            num[b, :, h] = mask.sum(1).double()
    return out, lse, pv, mag, num


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("ctx,window,first", [
    (1000, 600, 0), (1000, 600, 37), (1000, 500, 0), (1000, 488, 5), (511, 3, 0), (513, 4, 0), (520, None, 0), (TOP, None, 3),
    (TOP, 1, 9), (TOP, 1, 0), (TOP, 4096, 0), (TOP, TOP, 0), (TOP, TOP - 100, 1), ((1 << 30) + 700, 1 << 30, 0),
    ((1 << 30) + 700, (1 << 30) + 500, 2), ((1 << 30) + 700, (1 << 30) - 1, 0), (1 << 30, TOP, 0), ((3 << 29) + 5, (1 << 30) + 7, 66)])
def test_positions_past_the_table(form, page, ctx, window, first):
    """A table of 512 rows, beside a sequence that ends in it."""
    dtype, fp8, S, Hq, Hkv, D, Dv, mla = FORMS[form]
    c = _case(dtype, fp8, S=S, ctx=(512 - S, 200), Hq=Hq, Hkv=Hkv, D=D, Dv=Dv, page=page, mla=mla)
    c["ctx"] = torch.tensor([ctx, 200], dtype=torch.int32, device=DEV)
    for sink in (None, torch.randn(Hq, device=DEV)):
        got = _run(c, window=window, first=first, attn_sink=sink)
        ref.check(got, _want(c, [ctx, 200], window, first, sink), D, dtype, 2.0 ** -8 if dtype == BF else 0.0)
    long = dict(c, ctx=torch.tensor([ctx, 200], dtype=torch.int64, device=DEV))
    again = _run(long, window=window, first=first, attn_sink=sink)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
