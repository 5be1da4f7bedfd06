"""int64 ids and lengths that do not fit 32 bits: they are outside of every pool and
table, and stay so on the way to the kernels.  CPU only (what the kernels do with
ids outside is tested with them)."""
import ctypes

import torch

import ops_amd
from ops_amd import _host
from tests.host_calls import launches  # noqa: F401

WIDE = [1 << 31, 1 << 32, (1 << 32) + 3, (1 << 40) + 1, (1 << 63) - 1]
LOW = [-(1 << 31) - 1, -(1 << 32), -(1 << 32) + 2, -(1 << 63)]


def _read(address, n):
    return list((ctypes.c_int32 * n).from_address(address))


def test_int32_keeps_ids_outside():
    t = torch.tensor(WIDE + LOW + [-1, 0, 7, (1 << 31) - 1])
    assert _host.int32(t).tolist() == [(1 << 31) - 1] * len(WIDE) + [-(1 << 31)] * len(LOW) + [-1, 0, 7, (1 << 31) - 1]
    assert _host.int32(t.int()[-4:]).tolist() == [-1, 0, 7, (1 << 31) - 1]


def test_ids_and_lengths_of_the_calls(launches, monkeypatch):  # noqa: F811
    from ops_amd import cache, rope, tree
    seen = {}

    def call(device, fn, *args):  # (read while the call holds them)
        a = getattr(args[0], "_obj", None)
        if fn == "sfa_tree_fwd":
            seen[fn] = _read(a.ctx_lens, 2) + _read(a.tree_lens, 2) + _read(args[1]._obj.block_table, 4)
        elif fn == "sfa_rope_fwd":
            seen[fn] = _read(args[1]._obj.block_table, 4)
        elif fn == "sfa_cache_keep_path":
            seen[fn] = _read(args[1], 2) + _read(args[2], 2 * args[4])
        else:
            seen[fn] = _read(args[1], 2) + (_read(a.kv_lens, 2) if fn == "sfa_cache_extend" else _read(args[2], 2))

    for m in (cache, rope, tree):
        monkeypatch.setattr(m, "call", call)
    t = lambda *x: torch.tensor(x, dtype=torch.int64)  # noqa: E731
    wide, low, top = (1 << 32) + 1, -(1 << 32) + 1, (1 << 31) - 1
    pool = torch.zeros(4, 16, 1, 64)
    x, pos = torch.zeros(2, 3, 1, 64), torch.arange(3)
    bt, ids = t(wide, 0, low, 1).view(2, 2), t(wide, low)
    cut, cut_bt = [top, -(1 << 31)], [top, 0, -(1 << 31), 1]
    ops_amd.tree_attention_paged(x, pool, pool, bt, ids, torch.ones(2, 3, dtype=torch.int64), ids)
    ops_amd.qk_norm_rope_append(None, x, None, pool, None, bt, pos, pos, ops_amd.rope_frequencies(64))
    bt32, refs, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    ops_amd.cache_copy_pages([pool], ids, ids)
    ops_amd.cache_fork(bt32, refs, lens, ids, ids, [pool])
    ops_amd.cache_free(bt32, refs, ids, ids, page_size=16)
    ops_amd.cache_extend(bt32, refs, ids, ids, 16)
    ops_amd.cache_keep_path([pool], bt32, ids, bt)
    assert seen == {"sfa_tree_fwd": cut + cut + cut_bt, "sfa_rope_fwd": cut_bt, "sfa_cache_copy": cut + cut,
                    "sfa_cache_fork": cut + cut, "sfa_cache_free": cut + cut, "sfa_cache_extend": cut + cut,
                    "sfa_cache_keep_path": cut + cut_bt}
