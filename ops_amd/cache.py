"""Pages of a paged KV cache on MI355X: mapping, forking, freeing, compacting
and copying them, all on the device, and reading their rows back.

The state is the caller's: ``block_table`` int32 ``[B, max_pages]`` (the page of
each sequence's i-th run of ``page_size`` rows, -1: none) as the paged forwards
read it, and ``ref_counts`` int32 ``[num_pages]``, the number of table entries
that map a page.  A page is free iff its count is 0, and a call that takes
pages takes the lowest free ones, so results do not depend on timing.
``caches`` is a list of page pools ``[num_pages, page_size, ...]`` of any type
(each layer's K and V), each page contiguous.  The calls change the state in
place, never come back to the host, and can be captured in a graph.

The reference has no cache (lilac-me/ops SFA.py:88: one contiguous ``kv``).
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Sequence

import torch

from . import _lib
from ._host import (DTYPES, call, check_pool, check_scales, count32, int32, int_vec, kv_pages, need_gpu, strides4, table,
                    written)

__all__ = ["cache_copy_pages", "cache_fork", "cache_free", "cache_extend", "cache_compact", "cache_keep_path", "cache_read"]

_CACHE = struct.Struct("@P6iPqPP")
assert _CACHE.size == ctypes.sizeof(_lib.Cache)
_READ = struct.Struct("@6i" + 2 * "P3q" + "2P" + "P3q" + "i4x")
assert _READ.size == ctypes.sizeof(_lib.CacheReadArgs)


def _state(name: str, t: torch.Tensor, dim: int, device) -> None:
    """State that is changed in place: int32, unit stride, as it is."""
    need_gpu(name, t, device)
    if t.dtype != torch.int32 or t.dim() != dim or (t.numel() and t.stride(-1) != 1):
        raise ValueError(f"{name} must be a {dim}-D int32 tensor with unit stride (changed in place), got {t.dtype} "
                         f"{tuple(t.shape)}")
    written(t)


def _pools(caches: Sequence[torch.Tensor], device=None):
    """(packed sfa_cache_pool array, count, num_pages, page_size, device)."""
    if isinstance(caches, torch.Tensor):
        caches = [caches]
    if len(caches) == 0:
        raise ValueError("caches is empty")
    c0 = caches[0]
    if c0.dim() < 2:
        raise ValueError(f"a cache must be [num_pages, page_size, ...], got {tuple(c0.shape)}")
    need_gpu("caches", c0, device)
    num_pages, page_size, device = c0.shape[0], c0.shape[1], c0.device
    if page_size <= 0 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two, got {page_size}")
    vals = []
    for c in caches:
        if c.dim() < 2 or c.shape[0] != num_pages or c.shape[1] != page_size or c.device != device or c.numel() == 0:
            raise ValueError(f"caches must be [{num_pages}, {page_size}, ...] pools on {device}, got {tuple(c.shape)} on "
                             f"{c.device}")
        if not (c.is_contiguous() or c[0].is_contiguous()):
            raise ValueError("each page of a cache must be contiguous")
        written(c)
        e = c.element_size()
        vals += (c.data_ptr(), c.stride(0) * e, c.numel() // num_pages * e)
    if len(set(vals[::3])) != len(caches):
        raise ValueError("a cache is listed twice")
    return struct.pack(f"@{len(vals)}q", *vals), len(caches), num_pages, page_size, device


def _cache(pools, npools, num_pages, page_size, block_table=None, ref_counts=None, kv_lens=None):
    """sfa_cache; ``pools`` (bytes or None) must outlive the call."""
    buf = None if pools is None else ctypes.c_char_p(pools)
    bt = block_table
    try:
        a = _lib.Cache.from_buffer_copy(_CACHE.pack(
            0 if buf is None else ctypes.cast(buf, ctypes.c_void_p).value, npools, 0 if bt is None else bt.shape[0],
            0 if bt is None else bt.shape[1], page_size, num_pages, 0, 0 if bt is None else bt.data_ptr(),
            0 if bt is None else bt.stride(0), 0 if ref_counts is None else ref_counts.data_ptr(),
            0 if kv_lens is None else kv_lens.data_ptr()))
    except (struct.error, OverflowError) as e:
        raise ValueError(f"the call's arguments do not fit the kernels' interface: {e}") from None
    return a, buf


def _ws(lib, a, n, device):
    size = lib.sfa_cache_workspace_size(ctypes.byref(a), n)
    buf = torch.empty(max(size, 1), dtype=torch.uint8, device=device)
    return buf, buf.data_ptr(), size


def _check_refs(ref_counts, num_pages, device):
    _state("ref_counts", ref_counts, 1, device)
    if ref_counts.shape[0] != num_pages:
        raise ValueError(f"ref_counts must be [{num_pages}], got {tuple(ref_counts.shape)}")


def cache_copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Page ``src[i]`` copied to page ``dst[i]`` in every cache.  A pair is left
    out if either page is outside the pool, if a later pair has its destination,
    or if its destination is the source of another pair."""
    pools, n, num_pages, page_size, dev = _pools(caches)
    src = int_vec("src", src, src.shape[0] if src.dim() else 0, dev)
    dst = int_vec("dst", dst, src.shape[0], dev)
    if src.shape[0] == 0:
        return
    lib = _lib.load()
    a, keep = _cache(pools, n, num_pages, page_size)
    w, wp, size = _ws(lib, a, src.shape[0], dev)
    call(dev, lib.sfa_cache_copy, ctypes.byref(a), src.data_ptr(), dst.data_ptr(), src.shape[0], wp, size)


def cache_fork(block_table: torch.Tensor, ref_counts: torch.Tensor, kv_lens: torch.Tensor, parents: torch.Tensor,
               children: torch.Tensor, caches: Sequence[torch.Tensor]) -> torch.Tensor:
    """Row ``children[i]`` of the table becomes a fork of row ``parents[i]``: the
    whole pages of its ``kv_lens`` rows are shared, the rows of the last one,
    filled in part, are copied to a free page in every cache, and
    ``kv_lens[child] = kv_lens[parent]``.  Returns ``ok`` int32 ``[n]``: 0, with
    nothing written, for a pair with a row outside the table, whose child an
    earlier pair has or any pair has as its parent, or that finds no free page.
    Pages the child's row still maps are not freed: :func:`cache_free` first."""
    pools, n, num_pages, page_size, dev = _pools(caches)
    _state("block_table", block_table, 2, dev)
    _check_refs(ref_counts, num_pages, dev)
    _state("kv_lens", kv_lens, 1, dev)
    if kv_lens.shape[0] != block_table.shape[0]:
        raise ValueError(f"kv_lens must be [{block_table.shape[0]}], got {tuple(kv_lens.shape)}")
    parents = int_vec("parents", parents, parents.shape[0] if parents.dim() else 0, dev)
    children = int_vec("children", children, parents.shape[0], dev)
    ok = torch.empty(parents.shape[0], dtype=torch.int32, device=dev)
    if parents.shape[0] == 0:
        return ok
    lib = _lib.load()
    a, keep = _cache(pools, n, num_pages, page_size, block_table, ref_counts, kv_lens)
    w, wp, size = _ws(lib, a, parents.shape[0], dev)
    call(dev, lib.sfa_cache_fork, ctypes.byref(a), parents.data_ptr(), children.data_ptr(), parents.shape[0],
         ok.data_ptr(), wp, size)
    return ok


def cache_free(block_table: torch.Tensor, ref_counts: torch.Tensor, rows: torch.Tensor,
               keep_lens: Optional[torch.Tensor] = None, page_size: Optional[int] = None) -> None:
    """The entries of the table's ``rows`` become -1 and their pages lose a
    reference; with ``keep_lens`` ``[n]`` (and ``page_size``) each row keeps the
    pages of its first ``keep_lens[i]`` rows, e.g. after a draft is rejected.  Rows
    outside the table are left out, a row listed twice is freed once."""
    _state("block_table", block_table, 2, None)
    dev = block_table.device
    _state("ref_counts", ref_counts, 1, dev)
    rows = int_vec("rows", rows, rows.shape[0] if rows.dim() else 0, dev)
    if keep_lens is not None:
        if page_size is None:
            raise ValueError("keep_lens needs the page_size")
        keep_lens = int_vec("keep_lens", keep_lens, rows.shape[0], dev)
    if rows.shape[0] == 0 or block_table.numel() == 0:
        return
    lib = _lib.load()
    a, keep = _cache(None, 0, ref_counts.shape[0], 1 if page_size is None else int(page_size), block_table, ref_counts)
    call(dev, lib.sfa_cache_free, ctypes.byref(a), rows.data_ptr(), 0 if keep_lens is None else keep_lens.data_ptr(),
         rows.shape[0])


def cache_extend(block_table: torch.Tensor, ref_counts: torch.Tensor, kv_lens: torch.Tensor, new_lens: torch.Tensor,
                 page_size: int) -> torch.Tensor:
    """Free pages mapped for the rows ``kv_lens[b] .. new_lens[b] - 1`` of every
    sequence that has none there: all that a sequence needs or none, in order of
    b while they last.  Returns ``ok`` int32 ``[B]`` (0: it did not get them, or its
    rows do not fit the table; 1 also for a sequence that needs none);
    ``kv_lens`` is left to the caller."""
    _state("block_table", block_table, 2, None)
    dev, B = block_table.device, block_table.shape[0]
    _state("ref_counts", ref_counts, 1, dev)
    kv_lens, new_lens = int_vec("kv_lens", kv_lens, B, dev), int_vec("new_lens", new_lens, B, dev)
    ok = torch.empty(B, dtype=torch.int32, device=dev)
    if B == 0:
        return ok
    lib = _lib.load()
    a, keep = _cache(None, 0, ref_counts.shape[0], int(page_size), block_table, ref_counts, kv_lens)
    w, wp, size = _ws(lib, a, 0, dev)
    call(dev, lib.sfa_cache_extend, ctypes.byref(a), new_lens.data_ptr(), ok.data_ptr(), wp, size)
    return ok


def cache_compact(block_table: torch.Tensor, ref_counts: torch.Tensor, caches: Sequence[torch.Tensor]) -> torch.Tensor:
    """The pages in use moved, in order, to the free ids at the low end of every
    cache, the table and the counts with them.  Returns ``used`` int32 ``[1]``:
    afterwards the pages in use are exactly ``0 .. used - 1``."""
    pools, n, num_pages, page_size, dev = _pools(caches)
    _state("block_table", block_table, 2, dev)
    _check_refs(ref_counts, num_pages, dev)
    used = torch.empty(1, dtype=torch.int32, device=dev)
    lib = _lib.load()
    a, keep = _cache(pools, n, num_pages, page_size, block_table, ref_counts)
    w, wp, size = _ws(lib, a, 0, dev)
    call(dev, lib.sfa_cache_compact, ctypes.byref(a), used.data_ptr(), wp, size)
    return used


def cache_keep_path(caches: Sequence[torch.Tensor], block_table: torch.Tensor, ctx_lens: torch.Tensor,
                    path: torch.Tensor) -> None:
    """After a drafted tree is verified: row ``ctx_lens[b] + i`` of every cache
    becomes what row ``ctx_lens[b] + path[b, i]`` was (``path`` int32 ``[B, n]``, ``n
    <= 64``: the accepted nodes, in order; negative entries leave their row).  All
    rows are read before any is written.  The rows must lie on pages that no
    other sequence maps, which holds for everything behind a fork's context."""
    pools, n, num_pages, page_size, dev = _pools(caches)
    _state("block_table", block_table, 2, dev)
    B = block_table.shape[0]
    ctx_lens = int_vec("ctx_lens", ctx_lens, B, dev)
    need_gpu("path", path, dev)
    if path.dim() != 2 or path.shape[0] != B or path.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"path must be an integer [{B}, n] tensor, got {path.dtype} {tuple(path.shape)}")
    path = path if path.dtype == torch.int32 and (path.numel() == 0 or path.stride(1) == 1) \
        else int32(path).contiguous()
    if B == 0 or path.shape[1] == 0:
        return
    lib = _lib.load()
    a, keep = _cache(pools, n, num_pages, page_size, block_table)
    call(dev, lib.sfa_cache_keep_path, ctypes.byref(a), ctx_lens.data_ptr(), path.data_ptr(), path.stride(0),
         path.shape[1])


def cache_read(cache: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, length: int,
               starts: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None,
               dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The rows of a cache ``[num_pages, page_size, H, D]`` in order, ``[B, length, H,
    D]``: row ``i`` of sequence ``b`` is its row ``starts[b] + i`` (None: from 0), zeros
    past ``lens[b]`` and on unmapped pages.  What an e4m3 cache's bytes stand for,
    with its exponent bytes ``scales``, is exact in bfloat16 and float32
    (``dtype``; None: the cache's own, bfloat16 for e4m3, or ``out``'s).  ``out`` may be
    preallocated (unit feature stride, not part of the cache).  No gradient."""
    if cache.requires_grad and torch.is_grad_enabled():
        raise ValueError("reading a cache records no gradient: call it under torch.no_grad()")
    need_gpu("cache", cache)
    dev = cache.device
    check_pool("cache", cache, dev)
    fp8 = cache.dtype == torch.float8_e4m3fn
    if not fp8 and cache.dtype not in DTYPES:
        raise ValueError(f"unsupported cache dtype {cache.dtype}; expected bfloat16, float32 or float8_e4m3fn")
    if fp8:
        check_scales("scales", scales, cache, dev)
    elif scales is not None:
        raise ValueError("scales are those of an e4m3 cache")
    num_pages, page_size, H, D = cache.shape
    if cache.stride(3) != 1:
        raise ValueError("the cache needs a unit feature stride")
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [B, max_pages], got {tuple(block_table.shape)}")
    B, N = block_table.shape[0], count32("length", length, 0)
    bt = table(block_table, B, dev)
    lens = int_vec("lens", lens, B, dev)
    if starts is not None:
        starts = int_vec("starts", starts, B, dev)
    if dtype is None:
        dtype = out.dtype if out is not None else torch.bfloat16 if fp8 else cache.dtype
    if dtype not in DTYPES:
        raise ValueError(f"unsupported dtype {dtype}; expected bfloat16 or float32")
    if out is None:
        out = torch.empty((B, N, H, D), dtype=dtype, device=dev)
    elif tuple(out.shape) != (B, N, H, D) or out.dtype != dtype or out.device != dev or (out.numel() and out.stride(3) != 1):
        raise ValueError(f"out must be a {[B, N, H, D]} {dtype} tensor on {dev} with a unit feature stride")
    written(out)
    if out.numel() == 0:
        return out
    if num_pages == 0 or bt.shape[1] == 0:
        return out.zero_()
    try:
        a = _lib.CacheReadArgs.from_buffer_copy(_READ.pack(
            DTYPES[dtype], _lib.SFA_DTYPE_FP8_E4M3 if fp8 else DTYPES[cache.dtype], B, N, H, D, *strides4(cache),
            *strides4(scales), 0 if starts is None else starts.data_ptr(), lens.data_ptr(), *strides4(out), 0))
    except (struct.error, OverflowError) as e:
        raise ValueError(f"the call's arguments do not fit the kernels' interface: {e}") from None
    pg = kv_pages(bt, B, num_pages, page_size, dev)
    call(dev, _lib.load().sfa_cache_read, ctypes.byref(a), ctypes.byref(pg))
    return out
