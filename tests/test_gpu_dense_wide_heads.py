"""Gradients of dense attention with heads of more than 128 dims, whose dq several
workgroups make."""
import pytest
import torch

from tests.test_gpu_window import BF, F32, _check, _leaves, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D,Dv,S", [(192, 128, 1500), (300, 300, 1100), (576, 512, 600)])
def test_equal_calls_give_equal_bits(dtype, D, Dv, S):
    """Some thousands of workgroups: those of a row's dims run at different times."""
    x = _leaves(dtype, B=2, S=S, Hq=16, Hkv=4, D=D, Dv=Dv)
    a = _run(*x, window=700, first=4)
    for _ in range(3):
        b = _run(*x, window=700, first=4)
        assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_padded_batch_with_a_gradient_of_the_lse(dtype):
    x = _leaves(dtype, B=2, S=150, Hq=8, Hkv=2, D=300, Dv=200)
    lens = torch.tensor([150, 47], dtype=torch.int32, device="cuda")
    _check(x, lens=lens, dlse=torch.randn(2, 150, 8, device="cuda"), window=60, first=3)
