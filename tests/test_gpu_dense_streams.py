"""Dense attention and the 8-bit cache on another stream than the default one: what they read
is there only once earlier work of that stream is done."""
import math

import pytest
import torch

import ops_amd
from tests import dense_ref as ref
from tests.test_gpu_dense import BF, DEV, F8, _run
from tests.test_gpu_dense_calls import CASES, _case
from tests.test_gpu_window import _leaves
from tests.test_gpu_window import _run as _run_window

pytestmark = pytest.mark.gpu


def _late(tensors, call):
    """call() on a stream where the tensors get their values behind long products; before, and
    for every other stream, they are NaN (bytes: 255)."""
    real = [t.clone() for t in tensors]
    for t in tensors:
        t.fill_(255 if t.dtype == torch.uint8 else math.nan)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x = torch.randn(4096, 4096, device=DEV)
        for _ in range(30):
            x = torch.tanh(x @ x)
        for t, r in zip(tensors, real):
            t.copy_(r)
        got = call()
        late = not side.query()  # (the products are still running: the call did not wait for them)
    side.synchronize()
    assert late
    return got


@pytest.mark.parametrize("name", list(CASES))
def test_chunk(name):
    c = _case(**CASES[name])
    want = [t.clone() for t in _run(c)]
    got = _late([c["q"]], lambda: _run(c))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("D", [64, 128, 96, 192])
def test_training_step(D):
    x = _leaves(BF, B=1, S=200, Hq=8, Hkv=2, D=D)
    want = [t.clone() for t in _run_window(*x, window=70, first=2)]
    got = _late([x[0], x[3]], lambda: _run_window(*x, window=70, first=2))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_append_and_read():
    g = torch.Generator(device=DEV).manual_seed(4)
    B, S, H, D, page = 2, 40, 2, 128, 16
    k, v = (torch.randn(B, S, H, D, generator=g, device=DEV).to(BF) for _ in range(2))
    bt = ref.table([S] * B, page, 8, 0)
    lens = torch.full((B,), S, dtype=torch.int32, device=DEV)
    slots, freq = torch.arange(S, device=DEV), ops_amd.rope_frequencies(D, device=DEV)

    def call():
        kc, vc = (torch.zeros(8, page, H, D, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2))
        ks, vs = (torch.zeros(8, page, H, dtype=torch.uint8, device=DEV) for _ in range(2))
        ops_amd.qk_norm_rope_append(None, k, v, kc, vc, bt, slots, slots, freq, k_scales=ks, v_scales=vs)
        return [ops_amd.cache_read(c, bt, lens, S, scales=s) for c, s in ((kc, ks), (vc, vs))]
    want = [t.clone() for t in call()]
    got = _late([k, v], call)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = torch.randn(8, page, H, D, generator=g, device=DEV).to(BF)
    want = ops_amd.cache_read(x, bt, lens, S).clone()
    assert torch.equal(_late([x], lambda: ops_amd.cache_read(x, bt, lens, S)), want)
