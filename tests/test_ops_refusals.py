"""Calls of the operators around the attention that the host layer refuses, with
the GPU's checks passed by CPU tensors.  CPU only."""
import pytest
import torch

import ops_amd
from tests.host_calls import launches  # noqa: F401


def test_append_without_k_rows(launches):  # noqa: F811
    """No launch would turn q: its memory would be returned as it was allocated."""
    q, k, pool = torch.randn(2, 3, 4, 64), torch.randn(2, 3, 0, 64), torch.randn(9, 16, 0, 64)
    pos, bt = torch.arange(3), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="needs k rows"):
        ops_amd.qk_norm_rope_append(q, k, None, pool, None, bt, pos, pos, ops_amd.rope_frequencies(64))
    empty = ops_amd.qk_norm_rope_append(q[:0], q[:0], None, torch.randn(9, 16, 4, 64), None, bt[:0], pos, pos,
                                        ops_amd.rope_frequencies(64))
    assert empty.shape == (0, 3, 4, 64) and launches == []
