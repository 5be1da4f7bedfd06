"""Gradients of dense attention with many first tokens beside a window: their key blocks,
which all rows see, are sums of several workgroups."""
import pytest
import torch

from tests.test_gpu_window import BF, F32, _check, _leaves, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,first", [(64, 700), (1, 1299), (200, 1290), (3, 1152), (1000, 1000)])
def test_many_first_tokens(dtype, D, window, first):
    x = _leaves(dtype, B=2, S=1300, Hq=8, Hkv=2, D=D)
    lens = torch.tensor([1300, 1181], dtype=torch.int32, device="cuda")
    _check(x, lens=lens, window=window, first=first)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (F32, 64)])
def test_masks_that_are_causal(dtype, D):
    """To the bit: a window or first tokens that reach every row change nothing."""
    x = _leaves(dtype, B=1, S=900, Hq=16, Hkv=2, D=D)
    want = _run(*x)
    for window, first in ((None, 50), (900, 0), (900, 64), (70, 900), (1, (1 << 31) - 1)):
        assert all(torch.equal(a, b) for a, b in zip(want, _run(*x, window=window, first=first))), (window, first)
