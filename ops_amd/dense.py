"""Dense attention on MI355X, whole or through a sliding window with the first
tokens visible: a chunk of new tokens over a paged cache (serving), and whole
sequences with a backward (training).

The reference attends to the rows that an index names (lilac-me/ops
SFA.py:483-587).  A model that calls it has layers without an index beside it:
those that see everything, those that see a window, and every layer while the
context is shorter than the top-k; :func:`chunk_attention_paged` and
:func:`window_attention` are these.

Layout BSHD, query head ``h`` reads kv head ``h // (Hq // Hkv)``.  A token at row
``p`` sees the rows ``j <= p`` with ``j < first`` or ``p - j < window``.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._host import (DTYPES, call, check_pool, check_scales, count32, int_vec, kv_pages, need_gpu, rows, strides4, table,
                    written)

__all__ = ["chunk_attention_paged", "window_attention"]

_FWD = "10if4x" + 5 * "P3q" + "3P" + 2 * "P3q" + "i4x"
_ARGS = struct.Struct("@" + _FWD)
_BWD_ARGS = struct.Struct("@" + _FWD + 4 * "P3q" + "2P" + "i4x")
assert _ARGS.size == ctypes.sizeof(_lib.DenseArgs) and _BWD_ARGS.size == ctypes.sizeof(_lib.DenseBwdArgs)


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _pack(fmt: struct.Struct, *values) -> bytes:
    try:
        return fmt.pack(*values)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"the call's arguments do not fit the kernels' interface: {e}") from None


def _options(window, first, sm_scale, Dqk):
    """(window, first, scale) as the kernels take them; window 0: none."""
    w = 0 if window is None else count32("window", window, 1)
    return w, count32("first", first, 0), 1.0 / math.sqrt(Dqk) if sm_scale is None else float(sm_scale)


def _sink(attn_sink, Hq, dev):
    if attn_sink is None:
        return None
    need_gpu("attn_sink", attn_sink, dev)
    if attn_sink.numel() != Hq or not attn_sink.dtype.is_floating_point:
        raise ValueError(f"attn_sink must be a floating-point [{Hq}] tensor, got {attn_sink.dtype} {tuple(attn_sink.shape)}")
    return attn_sink.detach().to(torch.float32).contiguous()


def chunk_attention_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                          ctx_lens: torch.Tensor, chunk_lens: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                          window: Optional[int] = None, first: int = 0, attn_sink: Optional[torch.Tensor] = None,
                          k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
                          out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None):
    """``(out, lse)`` of the tokens ``q`` ``[B, S, Hq, Dqk]`` (``S = 1``: a decode step)
    over the pages of a cache that already holds their own k and v rows
    (:func:`ops_amd.qk_norm_rope_append`).

    ``k_cache`` / ``v_cache`` / ``block_table`` as in :func:`ops_amd.sfa_forward_paged`.
    Token ``s`` of sequence ``b`` stands at row ``ctx_lens[b] + s`` and sees the rows up
    to it (``window``: the last ``window`` of them, itself among them, and the
    ``first`` rows of the sequence); rows on unmapped pages and past the table are not
    seen (a context may end behind it).  Tokens at or past ``chunk_lens[b]`` (None: S)
    are padding: zeros and ``lse = -inf``.  A token that sees nothing gives the same
    (with ``attn_sink`` ``[Hq]``, which adds ``exp(sink)`` to each denominator, the sink as
    its ``lse``).

    ``float8_e4m3fn`` caches with exponent bytes ``k_scales`` / ``v_scales``
    (:func:`ops_amd.qk_norm_rope_append`) are attended to as the values that they
    stand for; of e4m3 latent rows ``v_cache`` is a view of ``k_cache`` and
    ``v_scales`` may be left out.  ``out`` ``[B, S, Hq, Dv]`` in q's type and ``lse``
    ``[B, S, Hq]`` float32 may be preallocated (memory of their own).  No
    gradient: inputs that ask for one are refused outside of ``torch.no_grad()``."""
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad
                                    or (attn_sink is not None and attn_sink.requires_grad)):
        raise ValueError("the attention over a cache records no gradient: call it under torch.no_grad()")
    if q.dim() != 4:
        raise ValueError(f"q must be 4-D (BSHD), got shape {tuple(q.shape)}")
    need_gpu("q", q)
    dev = q.device
    if q.dtype not in DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}; expected bfloat16 or float32")
    check_pool("k_cache", k_cache, dev)
    check_pool("v_cache", v_cache, dev)
    B, S, Hq, Dqk = q.shape
    num_pages, page_size, Hkv, Dk = k_cache.shape
    Dv = v_cache.shape[3]
    if Dk != Dqk or tuple(v_cache.shape[:3]) != (num_pages, page_size, Hkv):
        raise ValueError(f"caches {tuple(k_cache.shape)}, {tuple(v_cache.shape)} do not match q {tuple(q.shape)}")
    fp8 = k_cache.dtype == torch.float8_e4m3fn
    if k_cache.dtype != v_cache.dtype or (not fp8 and k_cache.dtype != q.dtype):
        raise ValueError("the caches must share q's dtype, or both be float8_e4m3fn")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the caches need a unit feature stride")
    if fp8:
        check_scales("k_scales", k_scales, k_cache, dev)
        if v_scales is None and v_cache.data_ptr() == k_cache.data_ptr():
            v_scales = k_scales
        check_scales("v_scales", v_scales, v_cache, dev)
    elif k_scales is not None or v_scales is not None:
        raise ValueError("scales are those of float8_e4m3fn caches")
    ctx_lens = int_vec("ctx_lens", ctx_lens, B, dev)
    if chunk_lens is not None:
        chunk_lens = int_vec("chunk_lens", chunk_lens, B, dev)
    attn_sink = _sink(attn_sink, Hq, dev)
    w, first, scale = _options(window, first, sm_scale, Dqk)
    bt = table(block_table, B, dev)
    q = rows(q)
    if out is None:
        out = torch.empty((B, S, Hq, Dv), dtype=q.dtype, device=dev)
    elif tuple(out.shape) != (B, S, Hq, Dv) or out.dtype != q.dtype or out.device != dev or out.stride(3) != 1:
        raise ValueError(f"out must be a {[B, S, Hq, Dv]} {q.dtype} tensor on {dev} with a unit feature stride")
    if lse is None:
        lse = torch.empty((B, S, Hq), dtype=torch.float32, device=dev)
    elif tuple(lse.shape) != (B, S, Hq) or lse.dtype != torch.float32 or lse.device != dev:
        raise ValueError(f"lse must be a {[B, S, Hq]} float32 tensor on {dev}")
    written(out, lse)
    if B * S == 0:
        return out, lse
    dt = DTYPES[q.dtype]
    a = _lib.DenseArgs.from_buffer_copy(_pack(
        _ARGS, dt, _lib.SFA_DTYPE_FP8_E4M3 if fp8 else dt, B, S, Hq, Hkv, Dqk, Dv, w, first, scale, *strides4(q),
        *strides4(k_cache), *strides4(v_cache), *strides4(k_scales), *strides4(v_scales), ctx_lens.data_ptr(),
        _ptr(chunk_lens), _ptr(attn_sink), *strides4(out), *strides4(lse), 0))
    pg = kv_pages(bt, B, num_pages, page_size, dev)
    lib = _lib.load()
    ra, rp = ctypes.byref(a), ctypes.byref(pg)
    ws = lib.sfa_dense_fwd_workspace_size(ra, rp)
    wbuf = torch.empty(ws, dtype=torch.uint8, device=dev) if ws else None
    call(dev, lib.sfa_dense_fwd, ra, rp, _ptr(wbuf), ws)
    return out, lse


class _WindowAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, attn_sink, lens, window, first, scale):
        dev = q.device
        B, S, Hq, Dqk = q.shape
        Hkv, Dv = k.shape[2], v.shape[3]
        sink = _sink(attn_sink, Hq, dev)
        q, k, v = rows(q), rows(k), rows(v)
        out = torch.empty((B, S, Hq, Dv), dtype=q.dtype, device=dev)
        lse = torch.empty((B, S, Hq), dtype=torch.float32, device=dev)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, out, lse, sink, lens)
        ctx.opts = (window, first, scale)
        ctx.sink_like = None if attn_sink is None else (attn_sink.shape, attn_sink.dtype)
        if B * S:
            lib = _lib.load()
            a = _lib.DenseArgs.from_buffer_copy(_pack(_ARGS, *_values(q, k, v, out, lse, sink, lens, ctx.opts)))
            ws = lib.sfa_dense_fwd_workspace_size(ctypes.byref(a), None)
            wbuf = torch.empty(ws, dtype=torch.uint8, device=dev) if ws else None
            call(dev, lib.sfa_dense_fwd, ctypes.byref(a), None, _ptr(wbuf), ws)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlse):
        q, k, v, out, lse, sink, lens = ctx.saved_tensors
        if dout is None and dlse is None:
            return (None,) * 8
        dev = q.device
        dout = torch.zeros_like(out) if dout is None else rows(dout)
        if dlse is not None:  # (lse is contiguous)
            dlse = dlse.to(torch.float32).contiguous()
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
        dsink = torch.empty_like(sink) if sink is not None and ctx.needs_input_grad[3] else None
        if q.shape[0] * q.shape[1]:
            lib = _lib.load()
            a = _lib.DenseBwdArgs.from_buffer_copy(_pack(
                _BWD_ARGS, *_values(q, k, v, out, lse, sink, lens, ctx.opts), *strides4(dout), *strides4(dq), *strides4(dk),
                *strides4(dv), _ptr(dlse), _ptr(dsink), 0))
            ws = lib.sfa_dense_bwd_workspace_size(ctypes.byref(a))
            wbuf = torch.empty(ws, dtype=torch.uint8, device=dev) if ws else None
            call(dev, lib.sfa_dense_bwd, ctypes.byref(a), _ptr(wbuf), ws)
        elif dsink is not None:
            dsink.zero_()
        if dsink is not None:
            dsink = dsink.view(ctx.sink_like[0]).to(ctx.sink_like[1])
        return dq, dk, dv, dsink, None, None, None, None


def _values(q, k, v, out, lse, sink, lens, opts):
    """The fields of ``sfa_dense_args`` without pages."""
    B, S, Hq, Dqk = q.shape
    dt = DTYPES[q.dtype]
    return (dt, dt, B, S, Hq, k.shape[2], Dqk, v.shape[3], *opts, *strides4(q), *strides4(k), *strides4(v), *strides4(None),
            *strides4(None), 0, _ptr(lens), _ptr(sink), *strides4(out), *strides4(lse), 0)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int] = None, first: int = 0,
                     sm_scale: Optional[float] = None, lens: Optional[torch.Tensor] = None,
                     attn_sink: Optional[torch.Tensor] = None):
    """Causal attention of whole sequences: ``(out, lse)`` of ``q`` ``[B, S, Hq, Dqk]``,
    ``k`` ``[B, S, Hkv, Dqk]``, ``v`` ``[B, S, Hkv, Dv]``.

    Token ``i`` sees the tokens ``j <= i`` with ``i - j < window`` (None: all of them)
    or ``j < first``.  ``lens`` ``[B]``: tokens at or past ``lens[b]`` are padding, whose
    values are not read; their ``out`` and gradients are zeros, their ``lse`` -inf.
    ``attn_sink`` ``[Hq]`` adds ``exp(sink)`` to each denominator.  Differentiable in q,
    k, v and the sink, through ``out`` and ``lse``; every gradient is summed in a fixed
    order, so that equal calls give equal bits."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-D (BSHD), got shape {tuple(t.shape)}")
    need_gpu("q", q)
    dev = q.device
    for name, t in (("k", k), ("v", v)):
        need_gpu(name, t, dev)
    if q.dtype not in DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must share bfloat16 or float32, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, S, Hq, Dqk = q.shape
    Hkv = k.shape[2]
    if tuple(k.shape) != (B, S, Hkv, Dqk) or tuple(v.shape[:3]) != (B, S, Hkv):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"Hq ({Hq}) must be a positive multiple of Hkv ({Hkv})")
    if lens is not None:
        lens = int_vec("lens", lens, B, dev)
    if attn_sink is not None:
        _sink(attn_sink, Hq, dev)
    return _WindowAttention.apply(q, k, v, attn_sink, lens, *_options(window, first, sm_scale, Dqk))
