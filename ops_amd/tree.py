"""Attention of a tree of drafted tokens over a paged cache on MI355X.

The verification step of speculative decoding: every sequence brings up to 64
drafted tokens, the nodes of a tree, whose k and v rows already lie in the
cache behind its context (:func:`ops_amd.qk_norm_rope_append`); each attends to
the whole context and to its own ancestors.  The reference has one query per
index row and no cache (lilac-me/ops SFA.py:483-587); this is the form without
index rows, for layers that attend to everything and for contexts no longer
than the top-k.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

import torch

from . import _lib
from ._host import DTYPES, call, check_pool, int_vec, kv_pages, need_gpu, rows, table, written

__all__ = ["tree_attention_paged"]

_ARGS = struct.Struct("@7if" + 3 * "P3q" + "P" + "P2q" + "2P" + 2 * "P3q" + "i4x")
assert _ARGS.size == ctypes.sizeof(_lib.TreeArgs)


def tree_attention_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                         ctx_lens: torch.Tensor, tree_mask: torch.Tensor, tree_lens: Optional[torch.Tensor] = None,
                         sm_scale: Optional[float] = None, attn_sink: Optional[torch.Tensor] = None,
                         out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None):
    """``(out, lse)`` of drafted tokens ``q`` ``[B, T, Hq, Dqk]``, ``T <= 64``.

    ``k_cache`` / ``v_cache`` / ``block_table`` as in
    :func:`ops_amd.sfa_forward_paged`.  Token t of sequence b sees the cache rows
    ``[0, ctx_lens[b])`` and the drafted rows ``ctx_lens[b] + j`` with bit j of
    ``tree_mask[b, t]`` (int64 ``[B, T]``: its ancestors and itself) and ``j <
    tree_lens[b]`` (None: T); rows on unmapped pages are not seen.  A token that
    sees nothing gives zeros and ``lse = -inf`` (with ``attn_sink`` ``[Hq]``, which
    adds ``exp(sink)`` to each denominator: the sink), a token past
    ``tree_lens[b]`` zeros and ``-inf``.  ``out`` ``[B, T, Hq, Dv]`` in q's type and
    ``lse`` ``[B, T, Hq]`` float32 may be preallocated (memory of their own).  No
    gradient: inputs that ask for one are refused outside of ``torch.no_grad()``."""
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad
                                    or (attn_sink is not None and attn_sink.requires_grad)):
        raise ValueError("the attention of drafted tokens records no gradient: call it under torch.no_grad()")
    if q.dim() != 4:
        raise ValueError(f"q must be 4-D (BSHD), got shape {tuple(q.shape)}")
    need_gpu("q", q)
    dev = q.device
    if q.dtype not in DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}; expected bfloat16 or float32")
    check_pool("k_cache", k_cache, dev)
    check_pool("v_cache", v_cache, dev)
    B, T, Hq, Dqk = q.shape
    num_pages, page_size, Hkv, Dk = k_cache.shape
    Dv = v_cache.shape[3]
    if Dk != Dqk or tuple(v_cache.shape[:3]) != (num_pages, page_size, Hkv):
        raise ValueError(f"caches {tuple(k_cache.shape)}, {tuple(v_cache.shape)} do not match q {tuple(q.shape)}")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError("q and the caches must share one dtype")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the caches need a unit feature stride")
    ctx_lens = int_vec("ctx_lens", ctx_lens, B, dev)
    need_gpu("tree_mask", tree_mask, dev)
    if tree_mask.dtype != torch.int64 or tuple(tree_mask.shape) != (B, T):
        raise ValueError(f"tree_mask must be int64 [{B}, {T}], got {tree_mask.dtype} {tuple(tree_mask.shape)}")
    if tree_lens is not None:
        tree_lens = int_vec("tree_lens", tree_lens, B, dev)
    if attn_sink is not None:
        need_gpu("attn_sink", attn_sink, dev)
        if attn_sink.numel() != Hq:
            raise ValueError("attn_sink must be a [Hq] tensor on q's device")
        attn_sink = attn_sink.to(torch.float32).contiguous()
    scale = 1.0 / math.sqrt(Dqk) if sm_scale is None else float(sm_scale)
    bt = table(block_table, B, dev)
    q = rows(q)
    if out is None:
        out = torch.empty((B, T, Hq, Dv), dtype=q.dtype, device=dev)
    elif tuple(out.shape) != (B, T, Hq, Dv) or out.dtype != q.dtype or out.device != dev or out.stride(3) != 1:
        raise ValueError(f"out must be a {[B, T, Hq, Dv]} {q.dtype} tensor on {dev} with a unit feature stride")
    if lse is None:
        lse = torch.empty((B, T, Hq), dtype=torch.float32, device=dev)
    elif tuple(lse.shape) != (B, T, Hq) or lse.dtype != torch.float32 or lse.device != dev:
        raise ValueError(f"lse must be a {[B, T, Hq]} float32 tensor on {dev}")
    written(out, lse)
    if B * T == 0:
        return out, lse
    lib = _lib.load()
    try:
        packed = _ARGS.pack(
            DTYPES[q.dtype], B, T, Hq, Hkv, Dqk, Dv, scale, q.data_ptr(), *q.stride()[:3], k_cache.data_ptr(),
            *k_cache.stride()[:3], v_cache.data_ptr(), *v_cache.stride()[:3], ctx_lens.data_ptr(), tree_mask.data_ptr(),
            *tree_mask.stride(), 0 if tree_lens is None else tree_lens.data_ptr(),
            0 if attn_sink is None else attn_sink.data_ptr(), out.data_ptr(), *out.stride()[:3], lse.data_ptr(),
            *lse.stride(), 0)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"the call's arguments do not fit the kernels' interface: {e}") from None
    a = _lib.TreeArgs.from_buffer_copy(packed)
    pg = kv_pages(bt, B, num_pages, page_size, dev)
    ra, rp = ctypes.byref(a), ctypes.byref(pg)
    ws = lib.sfa_tree_fwd_workspace_size(ra, rp)
    wbuf = torch.empty(ws, dtype=torch.uint8, device=dev) if ws else None
    call(dev, lib.sfa_tree_fwd, ra, rp, 0 if wbuf is None else wbuf.data_ptr(), ws)
    return out, lse
