"""Rotary positions and per-head norms of q and k on MI355X: the step before
the attention, in one pass over the rows.

The reference takes q and kv ready made (lilac-me/ops SFA.py:86-94); a layer
that calls it first normalises each head, turns part of it by its position
and, when serving, writes the k and v rows into the cache:

* :func:`rotary_embedding` turns one tensor (forward and backward);
* :func:`qk_norm_rope` norms and turns q and k (forward and backward, with the
  gradients of the norms' weights);
* :func:`qk_norm_rope_append` is its serving form: the k and v rows go straight
  into the pages of a cache.

Layout BSHD, as in :mod:`ops_amd.sfa`.  A norm covers the first
``len(weight)`` dims of a head (all of it, or the latent part of an MLA row);
the rotation covers ``2 * len(inv_freq)`` dims from ``rope_offset``, as pairs
``(i, i + R/2)`` or, ``interleaved``, ``(2i, 2i + 1)``.  Everything between the
load and the store is float32; angles are reduced in float64, so positions in
the millions keep their phase.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._host import DTYPES, call, check_pool, check_scales, int_rows, kv_pages, need_gpu, rows, strides4, table, written

__all__ = ["rope_frequencies", "rotary_embedding", "qk_norm_rope", "qk_norm_rope_append"]


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     original_length: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                     device=None) -> torch.Tensor:
    """The angles per position of a rotation of ``rotary_dim`` dims, float64
    ``[rotary_dim / 2]``: ``theta^(-2 i / rotary_dim)``, stretched for contexts
    ``factor`` times longer than trained on:

    ``linear``  all angles divided by ``factor``;
    ``ntk``     ``theta`` raised to ``theta * factor^(R / (R - 2))``: the fastest
                angle kept, the slowest divided by ``factor``;
    ``yarn``    by parts: angles that turn more than ``beta_fast`` times within
                ``original_length`` are kept, those that turn less than
                ``beta_slow`` times divided by ``factor``, a linear ramp over the
                index between (its score scale ``0.1 ln(factor) + 1`` is the
                caller's ``rope_scale``)."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if not theta > 1.0 or not factor > 0.0:
        raise ValueError("theta must be above 1 and factor positive")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be none, linear, ntk or yarn, got {scaling!r}")
    if scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs more than one pair")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    f = theta ** (-i / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if original_length <= 0:
            raise ValueError("yarn scaling needs the original_length of the training contexts")

        def index(turns):  # of the pair that turns so often within original_length
            return rotary_dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

        lo = max(0.0, math.floor(index(beta_fast)))
        # (past the last pair, up to the published bound, where even that one turns
        # more than beta_slow times: it then stays on the ramp)
        hi = min(rotary_dim - 1.0, math.ceil(index(beta_slow)))
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * (1.0 - ramp) + f / factor * ramp
    return f.to(device) if device is not None else f


_ARGS = struct.Struct("@15i2f" + "P2q" + "P" + 2 * "P3q" + "2P" + 4 * "P3q" + "P2q" + 2 * "P3q" + "2P" + "i4x")
assert _ARGS.size == ctypes.sizeof(_lib.RopeArgs)
_NONE = (0, 0, 0, 0)


def _t(t: Optional[torch.Tensor]) -> tuple:
    """Pointer and the three leading strides."""
    return _NONE if t is None else (t.data_ptr(), *t.stride()[:3])


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _weight(w: Optional[torch.Tensor], dtype: torch.dtype) -> Optional[torch.Tensor]:
    return w if w is None or (w.dtype == dtype and w.is_contiguous()) else w.detach().to(dtype).contiguous()


class _Call:
    """What the forward and the backward of one call share."""
    __slots__ = ("dtype", "B", "S", "D", "R", "off", "inter", "eps", "scale", "pos", "freq", "wq", "wk", "wdt")

    def __init__(self, x, positions, inv_freq, q_weight, k_weight, eps, rope_offset, interleaved, rope_scale):
        self.B, self.S, _, self.D = x.shape
        dev = x.device
        self.dtype = DTYPES[x.dtype]
        self.pos = int_rows("positions", positions, self.B, self.S, dev)
        if inv_freq.dim() != 1:
            raise ValueError(f"inv_freq must be one-dimensional, got {tuple(inv_freq.shape)}")
        need_gpu("inv_freq", inv_freq, dev)
        if inv_freq.dtype != torch.float64 or not inv_freq.is_contiguous():
            inv_freq = inv_freq.to(torch.float64).contiguous()
        self.freq = inv_freq
        self.R, self.off, self.inter = 2 * inv_freq.shape[0], int(rope_offset), int(bool(interleaved))
        self.eps, self.scale = float(eps), float(rope_scale)
        self.wdt = self.dtype
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is None:
                continue
            need_gpu(name, w, dev)
            if w.dim() != 1 or not 0 < w.shape[0] <= self.D:
                raise ValueError(f"{name} must be [n] with 0 < n <= {self.D}, got {tuple(w.shape)}")
            if w.dtype not in DTYPES:
                raise ValueError(f"unsupported dtype {w.dtype} of {name}")
            if w.dtype != x.dtype:
                self.wdt = _lib.SFA_DTYPE_F32
        wt = torch.float32 if self.wdt == _lib.SFA_DTYPE_F32 else x.dtype
        self.wq, self.wk = _weight(q_weight, wt), _weight(k_weight, wt)

    def args(self, q, k, q_out, k_out, v=None, v_out=None, slots=None, dq=None, dk=None, dwq=None, dwk=None):
        """``sfa_rope_args``; q_out None: no q, k_out None: no k."""
        wq, wk = self.wq if q_out is not None else None, self.wk if k_out is not None else None
        hq = 0 if q_out is None else (q if q is not None else q_out).shape[2]
        hk = 0 if k_out is None else (k if k is not None else k_out).shape[2]
        try:
            return _lib.RopeArgs.from_buffer_copy(_ARGS.pack(
                self.dtype, self.B, self.S, self.D, hq, hk, 0 if v is None else v.shape[3], self.R, self.off, self.inter,
                0 if wq is None else wq.shape[0], 0 if wk is None else wk.shape[0], self.wdt,
                self.pos.dtype == torch.int64, slots is not None and slots.dtype == torch.int64, self.eps, self.scale,
                self.pos.data_ptr(), *self.pos.stride(), self.freq.data_ptr(), *_t(q), *_t(k), _ptr(wq), _ptr(wk),
                *_t(q_out), *_t(k_out), *_t(v), *_t(v_out), _ptr(slots), *((0, 0) if slots is None else slots.stride()),
                *_t(dq), *_t(dk), _ptr(dwq), _ptr(dwk), 0))
        except (struct.error, OverflowError) as e:
            raise ValueError(f"the call's arguments do not fit the kernels' interface: {e}") from None


def _check_rows(name, x, like=None):
    if x.dim() != 4:
        raise ValueError(f"{name} must be 4-D (BSHD), got shape {tuple(x.shape)}")
    need_gpu(name, x, None if like is None else like.device)
    if x.dtype not in DTYPES:
        raise ValueError(f"unsupported dtype {x.dtype}; expected bfloat16 or float32")
    if like is not None and (x.dtype != like.dtype or x.shape[:2] != like.shape[:2]):
        raise ValueError(f"{name} {x.dtype} {tuple(x.shape)} does not match {like.dtype} {tuple(like.shape)}")


def _like(x):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


class _NormRope(torch.autograd.Function):
    """q (and k, or None) normed and turned."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, inv_freq, eps, rope_offset, interleaved, rope_scale):
        c = _Call(q, positions, inv_freq, q_weight, k_weight, eps, rope_offset, interleaved, rope_scale)
        q, k = rows(q), None if k is None else rows(k)
        qo, ko = _like(q), None if k is None else _like(k)
        if q.numel() + (0 if k is None else k.numel()) > 0:
            a = c.args(q, k, qo, ko)
            call(q.device, _lib.load().sfa_rope_fwd, ctypes.byref(a), None)
        # x itself is read again only where a norm has to be undone; the others
        # are saved for autograd's check that nobody has written them since
        ctx.save_for_backward(q if c.wq is not None else None, k if c.wk is not None else None, q_weight, k_weight,
                              c.pos, c.freq)
        ctx.call = c
        ctx.set_materialize_grads(False)
        return qo, ko

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, _, _ = ctx.saved_tensors
        need = ctx.needs_input_grad
        if not (need[0] or need[2]):
            gq = None
        if not (need[1] or need[3]):
            gk = None
        any_g = gq if gq is not None else gk
        if any_g is None:
            return (None,) * 10
        c = ctx.call
        gq, gk = None if gq is None else rows(gq), None if gk is None else rows(gk)
        dq, dk = None if gq is None else _like(gq), None if gk is None else _like(gk)
        dwq = None if gq is None or c.wq is None else torch.empty_like(c.wq) if gq.numel() else torch.zeros_like(c.wq)
        dwk = None if gk is None or c.wk is None else torch.empty_like(c.wk) if gk.numel() else torch.zeros_like(c.wk)
        if sum(g.numel() for g in (gq, gk) if g is not None) > 0:
            lib = _lib.load()
            a = c.args(q if gq is not None else None, k if gk is not None else None, gq, gk, dq=dq, dk=dk, dwq=dwq,
                       dwk=dwk)
            ws = lib.sfa_rope_bwd_workspace_size(ctypes.byref(a))
            wbuf = torch.empty(ws, dtype=torch.uint8, device=any_g.device) if ws else None
            call(any_g.device, lib.sfa_rope_bwd, ctypes.byref(a), _ptr(wbuf), ws)
        return (dq, dk, None if dwq is None else dwq.to(q_weight.dtype), None if dwk is None else dwk.to(k_weight.dtype),
                None, None, None, None, None, None)


def rotary_embedding(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, rope_offset: int = 0,
                     interleaved: bool = False, rope_scale: float = 1.0, out: Optional[torch.Tensor] = None):
    """``x`` ``[B, S, H, D]`` with its dims ``[rope_offset, rope_offset + 2 *
    len(inv_freq))`` turned by ``positions * inv_freq`` and multiplied by
    ``rope_scale``; ``positions`` ``[B, S]`` or ``[S]``, int32 or int64.

    Differentiable in ``x``.  With ``out`` (x's shape and type, unit feature
    stride; ``x`` itself turns it in place, any other memory must not overlap
    x's) there is no gradient."""
    _check_rows("x", x)
    if out is None:
        return _NormRope.apply(x, None, None, None, positions, inv_freq, 0.0, rope_offset, interleaved, rope_scale)[0]
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("out= records no gradient: call it under torch.no_grad() or without out")
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or (x.numel() and out.stride(-1) != 1):
        raise ValueError(f"out must be a {list(x.shape)} {x.dtype} tensor on {x.device} with a unit feature stride")
    c = _Call(x, positions, inv_freq, None, None, 0.0, rope_offset, interleaved, rope_scale)
    written(out)
    if x.numel() > 0:
        x = rows(x)  # (held until the launch, as everything a call reads)
        a = c.args(x, None, out, None)
        call(x.device, _lib.load().sfa_rope_fwd, ctypes.byref(a), None)
    return out


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 rope_offset: int = 0, interleaved: bool = False, rope_scale: float = 1.0):
    """Each head of ``q`` ``[B, S, Hq, D]`` and ``k`` ``[B, S, Hkv, D]`` divided by
    the root mean square of its first ``len(weight)`` dims (``eps`` added to the
    mean square) and scaled by the weight, then turned as in
    :func:`rotary_embedding`: ``(q_out, k_out)``.  A weight of None: no norm for
    that tensor.  Differentiable in q, k and the weights (bfloat16 or float32;
    their gradients are summed in float32 in a fixed order)."""
    _check_rows("q", q)
    _check_rows("k", k, q)
    if k.shape[3] != q.shape[3]:
        raise ValueError(f"q and k must have one head dim, got {q.shape[3]} and {k.shape[3]}")
    return _NormRope.apply(q, k, q_weight, k_weight, positions, inv_freq, eps, rope_offset, interleaved, rope_scale)


def qk_norm_rope_append(q: Optional[torch.Tensor], k: torch.Tensor, v: Optional[torch.Tensor], k_cache: torch.Tensor,
                        v_cache: Optional[torch.Tensor], block_table: torch.Tensor, slots: torch.Tensor,
                        positions: torch.Tensor, inv_freq: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                        k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, rope_offset: int = 0,
                        interleaved: bool = False, rope_scale: float = 1.0, out: Optional[torch.Tensor] = None,
                        k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None):
    """:func:`qk_norm_rope` for serving: returns the turned q (into ``out``, which
    may be ``q``; None without q), writes each token's k row to row
    ``slots[b, s]`` of sequence ``b`` in ``k_cache`` ``[num_pages, page_size, Hkv,
    D]`` and ``v`` ``[B, S, Hkv, Dv]``, unchanged, to ``v_cache``
    (``v = v_cache = None``: the v rows are part of the k rows, as for MLA).

    ``slots`` ``[B, S]`` or ``[S]`` are logical cache rows, apart from
    ``positions`` (drafted tokens of one depth share a position, not a row).
    A slot outside the table (e.g. -1: a padded token) or on an unmapped page is
    not written.  Slots of one call must differ; of two tokens with the same
    cache row, either's values may be left there.  No gradient.

    ``float8_e4m3fn`` pools take the rows quantised, each head's row on its own: its
    exponent ``e`` goes to ``k_scales`` / ``v_scales`` (uint8 or float8_e8m0fnu
    ``[num_pages, page_size, Hkv]``) and the row stands for its bytes' values times
    ``2^(e - 127)``, the smallest power of two, down to ``2^-111``, that leaves the
    row's largest finite magnitude at 448 or less; infinities become NaN."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, q_weight, k_weight)):
        raise ValueError("appending to a cache records no gradient: call it under torch.no_grad()")
    _check_rows("k", k)
    B, S, Hkv, D = k.shape
    dev = k.device
    if Hkv == 0:
        raise ValueError("append needs k rows, got k without heads (rotary_embedding or qk_norm_rope turn q alone)")
    if q is not None:
        _check_rows("q", q, k)
        if q.shape[3] != D:
            raise ValueError(f"q and k must have one head dim, got {q.shape[3]} and {D}")
    check_pool("k_cache", k_cache, dev)
    num_pages, page_size = k_cache.shape[:2]
    fp8 = k_cache.dtype == torch.float8_e4m3fn
    pool_type = torch.float8_e4m3fn if fp8 else k.dtype
    if tuple(k_cache.shape[2:]) != (Hkv, D) or k_cache.dtype != pool_type or k_cache.stride(3) != 1:
        raise ValueError(f"k_cache must be a [num_pages, page_size, {Hkv}, {D}] {k.dtype} or float8_e4m3fn pool with a unit "
                         "feature stride")
    if (v is None) != (v_cache is None):
        raise ValueError("v and v_cache go together")
    if v is not None:
        _check_rows("v", v, k)
        check_pool("v_cache", v_cache, dev)
        if v.shape[2] != Hkv or tuple(v_cache.shape) != (num_pages, page_size, Hkv, v.shape[3]) \
                or v_cache.dtype != pool_type or v_cache.stride(3) != 1:
            raise ValueError(f"v_cache must be a [{num_pages}, {page_size}, {Hkv}, {v.shape[3]}] {pool_type} pool with a "
                             "unit feature stride, v [B, S, Hkv, Dv]")
        v = rows(v)
    if fp8:
        check_scales("k_scales", k_scales, k_cache, dev)
        if v is not None:
            check_scales("v_scales", v_scales, v_cache, dev)
    if (k_scales is not None and not fp8) or (v_scales is not None and (v is None or not fp8)):
        raise ValueError("scales are those of float8_e4m3fn pools")
    c = _Call(k, positions, inv_freq, q_weight if q is not None else None, k_weight, eps, rope_offset, interleaved,
              rope_scale)
    bt = table(block_table, B, dev)
    slots = int_rows("slots", slots, B, S, dev)
    if out is not None and (q is None or out.shape != q.shape or out.dtype != q.dtype or out.device != dev
                            or (q.numel() and out.stride(-1) != 1)):
        raise ValueError("out must be a tensor like q with a unit feature stride")
    if q is not None:
        q = rows(q)
        out = _like(q) if out is None else out
    written(out, k_cache, v_cache, k_scales, v_scales)
    if k.numel() > 0:
        k = rows(k)
        a = c.args(q, k, out, k_cache, v, v_cache, slots)
        pg = kv_pages(bt, B, num_pages, page_size, dev)
        if fp8:
            sc = _lib.KvScales(*strides4(k_scales), *strides4(v_scales))
            call(dev, _lib.load().sfa_rope_append_fp8, ctypes.byref(a), ctypes.byref(pg), ctypes.byref(sc))
        else:
            call(dev, _lib.load().sfa_rope_fwd, ctypes.byref(a), ctypes.byref(pg))
    return out
