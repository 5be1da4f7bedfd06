"""The stretched frequencies ("yarn") against their closed form, pair by pair, for
training contexts short and long: past 2 pi theta beta_slow positions even the
slowest pair turns more than beta_slow times, and the ramp ends behind the last
pair.  CPU only."""
import math

import pytest
import torch

import ops_amd


def _closed(R, theta, factor, length, fast, slow):
    def index(turns):  # of the pair that turns so often within length
        return R * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))

    lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), R - 1)
    f = []
    for i in range(R // 2):
        ramp = min(max((i - lo) / (hi - lo if hi != lo else 0.001), 0.0), 1.0)
        a = theta ** (-2 * i / R)
        f.append(a * (1 - ramp) + a / factor * ramp)
    return torch.tensor(f, dtype=torch.float64)


@pytest.mark.parametrize("R,theta", [(64, 1e4), (128, 1e4), (64, 5e5), (32, 100.0)])
@pytest.mark.parametrize("length", [64, 4096, 65536, 131072, 1 << 20])
@pytest.mark.parametrize("factor", [1.0, 4.0, 32.0])
def test_yarn_pair_by_pair(R, theta, length, factor):
    fast, slow = 32.0, 1.0
    y = ops_amd.rope_frequencies(R, theta, "yarn", factor, length, fast, slow)
    # (a dozen float64 operations on each side)
    assert torch.allclose(y, _closed(R, theta, factor, length, fast, slow), rtol=1e-13, atol=0.0)
    p = ops_amd.rope_frequencies(R, theta)
    turns = length * p / (2 * math.pi)
    assert torch.equal(y[turns > 2 * fast], p[turns > 2 * fast])
    if factor > 1.0:  # nothing that turns more than `slow` times loses the whole factor
        assert bool((y[turns > slow] > p[turns > slow] / factor * (1 + 1e-12)).all())


def test_yarn_last_pair_of_a_long_training_context():
    """64 dims, theta 1e4, 131072 positions: the last pair turns 2.78 times, 9 / 13
    of the way down the ramp from pair 22 = floor(22.51) to 35 = ceil(34.55)."""
    y, p = ops_amd.rope_frequencies(64, 1e4, "yarn", 8.0, 131072), ops_amd.rope_frequencies(64, 1e4)
    lo = math.floor(64 * math.log(131072 / (64 * math.pi)) / (2 * math.log(1e4)))
    hi = math.ceil(64 * math.log(131072 / (2 * math.pi)) / (2 * math.log(1e4)))
    assert hi > 31  # behind the last pair
    ramp = (31 - lo) / (hi - lo)
    assert abs(float(y[31] / p[31]) - (1 - ramp + ramp / 8)) < 1e-13
