"""GPU tests of mapping pages when the pool runs out, against what each sequence
has to get, spelled out."""
import pytest
import torch

import ops_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("i64", [False, True])
def test_sequences_that_need_no_page_are_ok_behind_the_last_one(i64):
    """Three pages are free.  Sequence 0 takes one, 1 asks for three more than are
    left and gets none, 2 and 4 have the pages of their rows already (4 asks for
    fewer rows than it has), 3 needs one and comes too late, 5 does not fit."""
    bt = _i([[0, -1, -1, -1], [1, -1, -1, -1], [2, 3, -1, -1], [4, -1, -1, -1], [5, -1, -1, -1], [6, -1, -1, -1]])
    refs = _i([1, 1, 1, 1, 1, 1, 1, 0, 0, 0])
    lens, new = [16, 16, 20, 16, 9, 16], [17, 64, 32, 17, 3, 65]
    lens, new = (torch.tensor(x, dtype=torch.int64 if i64 else torch.int32, device=DEV) for x in (lens, new))
    ok = ops_amd.cache_extend(bt, refs, lens, new, 16)
    torch.cuda.synchronize()
    assert ok.tolist() == [1, 0, 1, 0, 1, 0]
    assert bt.tolist() == [[0, 7, -1, -1], [1, -1, -1, -1], [2, 3, -1, -1], [4, -1, -1, -1], [5, -1, -1, -1], [6, -1, -1, -1]]
    assert refs.tolist() == [1, 1, 1, 1, 1, 1, 1, 1, 0, 0]


def test_a_full_pool_still_serves_sequences_that_need_nothing():
    B = 300
    bt, refs = torch.arange(B, dtype=torch.int32, device=DEV)[:, None].repeat(1, 2), torch.ones(B, dtype=torch.int32, device=DEV)
    bt[:, 1] = -1
    lens = torch.full((B,), 5, dtype=torch.int32, device=DEV)
    new = torch.where(torch.arange(B, device=DEV) % 3 == 1, 17, 16)
    ok = ops_amd.cache_extend(bt, refs, lens, new, 16)
    torch.cuda.synchronize()
    assert ok.tolist() == [int(b % 3 != 1) for b in range(B)]
    assert bool((bt[:, 1] == -1).all()) and bool((refs == 1).all())
