"""Dense attention with scales far from 1 / sqrt(D)."""
import pytest
import torch

from tests import dense_ref as ref
from tests.test_gpu_window import BF, F32, _leaves, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 40, 192])
@pytest.mark.parametrize("scale", [1e-40, 1.2e-38, 1e-37, 2.0 ** -101, 2.0 ** -99, 1e-20, 1e-6, 0.3])
def test_gradients_at_any_scale(dtype, D, scale):
    """Where scale is tiny all weights of a row are equal, whatever the LSE divided by it is."""
    x = _leaves(dtype, B=2, S=90, D=D)
    got = _run(*x, window=50, first=3, sm_scale=scale)
    want = ref.window(*x[:4], None, 50, 3, x[4], None, scale, dtype, 2.0 ** -8 if dtype == BF else 0.0)
    # (dq and dk are products with scale: below float32's normal range 2^-126, which bf16 shares,
    # steps are absolute, 2^-133 in bf16; a few of them where the float32 sums and the result are there)
    want = [(y, e + (2.0 ** -131 if i in (2, 3) else 0.0)) for i, (y, e) in enumerate(want)]
    ref.check_all(got, want)
