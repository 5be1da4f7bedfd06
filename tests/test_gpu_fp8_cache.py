"""Rows quantised as they are written into a cache's pages, and read back, against
the formulas in float64."""
import math

import pytest
import torch

import ops_amd
from tests import dense_ref as ref
from tests import ops_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _pools(num, page, H, D):
    """An e4m3 pool and its exponents, filled with a pattern that must stay where nothing is written."""
    return (torch.full((num, page, H, D), 0x2a, dtype=torch.uint8, device=DEV).view(F8),
            torch.full((num, page, H), 99, dtype=torch.uint8, device=DEV))


def _row(pool, scales, bt, b, slot):
    ps = pool.shape[1]
    p = int(bt[b, slot // ps])
    return pool.view(torch.uint8)[p, slot % ps], scales[p, slot % ps]


def _near(pool, scales, x, rel):
    """The stored rows are x (float64, off by rel of its largest at most) rounded: half a step
    of e4m3 from it, under a scale that fits it."""
    e = scales.double()
    unit = torch.exp2(e - 127)[..., None]
    amax = x.abs().amax(-1)
    top = 448 * unit[..., 0]
    assert bool((amax <= top * (1 + rel)).all()) and bool(((e == 16) | (amax > top / 2 * (1 - rel))).all())
    y = pool.view(F8).double() * unit
    step = torch.exp2(torch.floor(torch.log2((x.abs() / unit).clamp(min=2.0 ** -6, max=448.0))) - 3) * unit
    # (next to a power of two the wider step is the one above)
    err = (y - x).abs() - (step / 2 * (1 + 2.0 ** -4 * 0) + rel * amax[..., None])
    assert float(err.max()) <= 0.0, float(err.max())


SHAPES = [  # heads, kv heads, D, Dv, rotary, offset, interleaved, k_norm
    (8, 2, 128, 128, 128, 0, False, 128), (4, 4, 64, 64, 64, 0, True, 64), (4, 1, 64, 64, 32, 0, False, 0),
    (4, 1, 576, 0, 64, 512, True, 512), (3, 3, 33, 17, 10, 3, False, 20), (2, 2, 96, 64, 96, 0, False, 96),
    (2, 1, 256, 256, 128, 64, True, 256), (1, 1, 1024, 1024, 64, 0, False, 1024), (4, 2, 40, 40, 0, 0, False, 0)]


@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[2]}-{s[3]}" for s in SHAPES])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 37])
def test_append(shape, dtype, S):
    Hq, H, D, Dv, R, off, inter, kn = shape
    g = torch.Generator(device=DEV).manual_seed(D + S)
    B, page = 3, 16
    q, k = torch.randn(B, S, Hq, D, generator=g, device=DEV).to(dtype), torch.randn(B, S, H, D, generator=g, device=DEV).to(dtype)
    k = k * torch.exp2(torch.randint(-20, 20, (B, S, H, 1), generator=g, device=DEV).float()).to(dtype)
    v = torch.randn(B, S, H, Dv, generator=g, device=DEV).to(dtype) if Dv else None
    wk = (1 + 0.1 * torch.randn(kn, generator=g, device=DEV)).to(dtype) if kn else None
    freq = ops_amd.rope_frequencies(R, device=DEV) if R else torch.zeros(0, dtype=torch.float64, device=DEV)
    bt = ref.table([60] * B, page, 4 * B + 2, S)
    slots = torch.stack([torch.randperm(60, generator=torch.Generator().manual_seed(b))[:S] for b in range(B)]).to(DEV)
    slots[1, 0] = -1  # a padded token
    if S > 3:
        slots[2, 3] = 10 ** 10
    bt[0, 2] = -1  # rows 32 .. 47 of sequence 0 go nowhere
    pos = slots.clamp(0, 60) * 1000
    (kc, ks), (vc, vs) = _pools(4 * B + 2, page, H, D), _pools(4 * B + 2, page, H, max(Dv, 1))
    before = kc.clone(), ks.clone()
    out = ops_amd.qk_norm_rope_append(q, k, v, kc, vc if Dv else None, bt, slots, pos, freq, None, wk, rope_offset=off, interleaved=inter,
                                      k_scales=ks, v_scales=vs if Dv else None)
    want_q = ops_ref.rotate(q.double(), pos, freq, off, inter)
    rel = 2.0 ** -19
    assert float(((out.double() - want_q).abs() - (ref.half(dtype) * want_q.abs() + rel * q.double().abs().amax())).max()) <= 0.0
    want = ops_ref.rotate(ops_ref.norm(k.double(), wk, 1e-6)[0], pos, freq, off, inter)
    wrote = torch.zeros(4 * B + 2, page, dtype=torch.bool, device=DEV)
    for b in range(B):
        for s in range(S):
            slot = int(slots[b, s])
            if not 0 <= slot < 64 or int(bt[b, slot // page]) < 0:
                continue
            wrote[int(bt[b, slot // page]), slot % page] = True
            # float32: the norm's sum of D squares and a few products; the turned row may be
            # smaller than the one it comes from
            x = want[b, s]
            slack = rel * float(ops_ref.norm(k.double(), wk, 1e-6)[0][b, s].abs().amax() / x.abs().amax())
            _near(*_row(kc, ks, bt, b, slot), x, max(rel, slack))
            if Dv:
                y, e = _row(vc, vs, bt, b, slot)
                bytes_, ee = ref.quantised(v[b, s])
                assert torch.equal(y, bytes_.view(torch.uint8)) and torch.equal(e, ee)
    assert torch.equal(kc.view(torch.uint8)[~wrote], before[0].view(torch.uint8)[~wrote]) and torch.equal(ks[~wrote], before[1][~wrote])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 72, 33, 576])
def test_every_rounding(dtype, D):
    """Without norm or rotation the bytes are the formula's own: ties, the ends of the range,
    zeros, subnormal steps, infinities, the largest and smallest rows."""
    g = torch.Generator(device=DEV).manual_seed(1)
    rows = [torch.randn(D, generator=g, device=DEV) * 2.0 ** e for e in (-126, -119, -100, -20, 0, 5, 100, 119)]
    rows += [torch.zeros(D, device=DEV), torch.full((D,), 448.0, device=DEV), torch.full((D,), 450.0, device=DEV)]
    rows += [torch.randint(-64, 65, (D,), generator=g, device=DEV) / 32.0 * 2.0 ** e for e in (-3, 0, 4)]  # ties
    rows += [torch.linspace(-448, 448, D, device=DEV), torch.randn(D, generator=g, device=DEV) * 2.0 ** -12]
    rows[-1][0] = 100.0  # all others below the smallest normal value of its scale
    x = torch.stack(rows).to(dtype)
    n = x.shape[0]
    bt = torch.arange(n, device=DEV, dtype=torch.int32).view(1, n)
    kc, ks = _pools(n, 1, 1, D)
    none = torch.zeros(0, dtype=torch.float64, device=DEV)
    slots = torch.arange(n, device=DEV)
    ops_amd.qk_norm_rope_append(None, x.view(1, n, 1, D), None, kc, None, bt, slots, slots, none, k_scales=ks)
    want, e = ref.quantised(x)
    assert torch.equal(ks.view(n), e)
    assert torch.equal(kc.view(n, D).float(), want.float())
    bad = x.clone()
    bad[:, 1], bad[:, 2], bad[:, 3] = math.inf, -math.inf, math.nan
    ops_amd.qk_norm_rope_append(None, bad.view(1, n, 1, D), None, kc, None, bt, slots, slots, none, k_scales=ks)
    fin = bad.clone()
    fin[:, 1:4] = 0.0
    want, e = ref.quantised(fin)
    got = kc.view(n, D).float()
    assert torch.equal(ks.view(n), e) and bool(torch.isnan(got[:, 1:4]).all())
    got[:, 1:4] = 0.0
    assert torch.equal(got, want.float())


@pytest.mark.parametrize("kind", ["e4m3", "e4m3-e8m0", "bf16", "f32"])
@pytest.mark.parametrize("H,D", [(2, 128), (1, 576), (3, 20), (1, 7), (8, 64)])
def test_read(kind, H, D):
    """Every row is the value it stands for, to the bit; rows that are not there are zeros."""
    g = torch.Generator(device=DEV).manual_seed(D)
    lens, page = [50, 0, 33, 64], 16
    num = 16
    bt = ref.table(lens, page, num, 0, extra=1)
    x = torch.randn(num, page, H, D, generator=g, device=DEV)
    scales = None
    if kind.startswith("e4m3"):
        x = x * torch.exp2(torch.randint(-60, 60, (num, page, H, 1), generator=g, device=DEV).float())
        x, scales = ref.quantised(x)
        scales[int(bt[0, 0]), 3] = 255
        scales = scales.view(torch.float8_e8m0fnu) if kind.endswith("e8m0") else scales
    else:
        x = x.to(BF if kind == "bf16" else F32)
    bt[3, 1] = -1
    bt[2, 0] = num
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    n[3] = 1000  # past the table
    for starts in (None, torch.tensor([7, 0, -2, 40], dtype=torch.int64, device=DEV)):
        for dtype in (None, BF, F32):
            N = 70
            got = ops_amd.cache_read(x, bt, n, N, starts, scales, dtype)
            assert got.dtype == (dtype or (BF if scales is not None else x.dtype)) and got.shape == (4, N, H, D)
            want = torch.zeros(4, N, H, D, dtype=torch.float64, device=DEV)
            for b in range(4):
                for i in range(N):
                    j = i + (0 if starts is None else int(starts[b]))
                    if 0 <= j < min(int(n[b]), bt.shape[1] * page) and 0 <= int(bt[b, j // page]) < num:
                        p = int(bt[b, j // page])
                        want[b, i] = ref.values(x[p, j % page], None if scales is None else scales[p, j % page])
            if scales is not None and starts is None:
                assert bool(torch.isnan(got[0, 3]).all())
            if scales is not None:
                at = 3 if starts is None else None
                if at is not None:
                    got[0, 3] = want[0, 3] = 0
                want = want.nan_to_num(0.0)
                got = got.nan_to_num(0.0)
            assert torch.equal(got, want.to(got.dtype))


def test_read_into_views():
    g = torch.Generator(device=DEV).manual_seed(5)
    x, s = ref.quantised(torch.randn(6, 8, 2, 64, generator=g, device=DEV))
    bt = ref.table([30], 8, 6, 0)
    n = torch.tensor([30], dtype=torch.int32, device=DEV)
    want = ops_amd.cache_read(x, bt, n, 30, scales=s)
    for off in (0, 1):
        out = torch.zeros(30, 1, 2, 72, dtype=F32, device=DEV).transpose(0, 1)[..., off:off + 64]
        assert ops_amd.cache_read(x, bt, n, 30, scales=s, out=out) is out
        assert torch.equal(out, want.float())
    assert ops_amd.cache_read(x, bt, n, 0, scales=s).shape == (1, 0, 2, 64)
    assert ops_amd.cache_read(x, bt[:0], n[:0], 5, scales=s).shape == (0, 5, 2, 64)


def test_written_read_and_attended():
    """A prompt and three decoded tokens through an 8-bit cache, as a program runs them: what
    is attended to is what is read back."""
    g = torch.Generator(device=DEV).manual_seed(9)
    B, Hq, H, D, page, P = 2, 8, 2, 128, 64, 150
    freq = ops_amd.rope_frequencies(D, device=DEV)
    w = torch.ones(D, dtype=BF, device=DEV)
    num = 8
    (kc, ks), (vc, vs) = _pools(num, page, H, D), _pools(num, page, H, D)
    bt = torch.full((B, 4), -1, dtype=torch.int32, device=DEV)
    refs, lens = torch.zeros(num, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    for step, S in enumerate((P, 1, 1, 1)):
        new = lens + S
        assert bool(ops_amd.cache_extend(bt, refs, lens, new, page).all())
        q, k, v = (torch.randn(B, S, h, D, generator=g, device=DEV).to(BF) for h in (Hq, H, H))
        slots = lens[:, None] + torch.arange(S, device=DEV)
        q = ops_amd.qk_norm_rope_append(q, k, v, kc, vc, bt, slots, slots, freq, w, w, k_scales=ks, v_scales=vs)
        got = ops_amd.chunk_attention_paged(q, kc, vc, bt, lens, window=100, first=4, k_scales=ks, v_scales=vs)
        L = P + step
        kr, vr = (ops_amd.cache_read(c, bt, new, L, scales=s) for c, s in ((kc, ks), (vc, vs)))
        flat = torch.arange(B, device=DEV, dtype=torch.int32).view(B, 1)
        pad = 256
        kp, vp = (torch.zeros(B, pad, H, D, dtype=BF, device=DEV) for _ in range(2))
        kp[:, :L], vp[:, :L] = kr, vr
        ref.check(got, ref.chunk(q, kp, vp, flat, lens, None, 100, 4), D, BF, 2.0 ** -8)
        plain = ops_amd.chunk_attention_paged(q, kp, vp, flat, lens, window=100, first=4)
        ref.check(plain, ref.chunk(q, kp, vp, flat, lens, None, 100, 4), D, BF, 2.0 ** -8)
        lens = new
    copy = [t.clone() for t in (kc.view(torch.uint8), ks)]
    ops_amd.cache_copy_pages([kc.view(torch.uint8), ks], bt[:1, 0].clone(), bt[1:2, 0].clone())
    assert torch.equal(kc.view(torch.uint8)[int(bt[1, 0])], copy[0][int(bt[0, 0])]) and torch.equal(ks[int(bt[1, 0])], copy[1][int(bt[0, 0])])
