"""What the host layers of the operators around the attention share: calls on
the current stream of the tensors' device, argument checks."""
from __future__ import annotations

import torch

from . import _lib

DTYPES = {torch.float32: _lib.SFA_DTYPE_F32, torch.bfloat16: _lib.SFA_DTYPE_BF16}
INTS = (torch.int32, torch.int64)


def call(device: torch.device, fn, *args) -> None:
    """``fn(*args, stream)`` with ``device`` (the tensors') the current device
    and its current stream; errors as exceptions."""
    i = device.index
    if torch._C._cuda_getDevice() == i:
        _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(i)))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(i)))


def need_gpu(name: str, t: torch.Tensor, device: torch.device = None) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (got device {t.device})")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device} (got {t.device})")


def written(*tensors) -> None:
    """The caller's tensors that a call is about to write: their elements must be
    distinct in memory, and autograd is told, so that a graph that has saved one
    raises instead of using what was written."""
    for t in tensors:
        if t is None:
            continue
        if 0 in t.stride() and any(st == 0 and n > 1 for n, st in zip(t.shape, t.stride())):
            raise ValueError(f"a tensor that is written must not be expanded (shape {tuple(t.shape)}, strides {t.stride()})")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("a tensor that is written must not require a gradient: call under torch.no_grad()")
        torch.autograd.graph.increment_version(t)


def rows(t: torch.Tensor) -> torch.Tensor:
    """The kernels need a unit stride on the feature dimension."""
    return t if t.stride(-1) == 1 else t.contiguous()


def int_rows(name: str, t: torch.Tensor, B: int, S: int, device: torch.device) -> torch.Tensor:
    """``[B, S]`` or ``[S]`` int32 / int64 as a ``[B, S]`` view (any strides)."""
    need_gpu(name, t, device)
    if t.dtype not in INTS:
        raise ValueError(f"{name} must be int32 or int64 (got {t.dtype})")
    if t.dim() == 1 and t.shape[0] == S:
        t = t.expand(B, S)
    if tuple(t.shape) != (B, S):
        raise ValueError(f"{name} must be [{B}, {S}] or [{S}], got {tuple(t.shape)}")
    return t


def int32(t: torch.Tensor) -> torch.Tensor:
    """int64 ids and lengths as int32.  Those past its range stay past every pool
    and table, which hold fewer than 2^31 rows: cut to 32 bits they would come
    back as page 0 or as a short length."""
    return t if t.dtype == torch.int32 else t.clamp(-1 << 31, (1 << 31) - 1).to(torch.int32)


def int_vec(name: str, t: torch.Tensor, n: int, device: torch.device) -> torch.Tensor:
    """A contiguous int32 ``[n]`` tensor."""
    need_gpu(name, t, device)
    if t.dtype not in INTS or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must be an integer [{n}] tensor, got {t.dtype} {tuple(t.shape)}")
    return t if t.dtype == torch.int32 and t.is_contiguous() else int32(t).contiguous()


def check_pool(name: str, t: torch.Tensor, device: torch.device) -> None:
    need_gpu(name, t, device)
    if t.dim() != 4:
        raise ValueError(f"{name} must be [num_pages, page_size, Hkv, D], got {tuple(t.shape)}")
    ps = t.shape[1]
    if ps <= 0 or ps & (ps - 1):
        raise ValueError(f"page_size must be a power of two, got {ps}")


def kv_pages(block_table: torch.Tensor, B: int, num_pages: int, page_size: int, device: torch.device) -> _lib.KvPages:
    """``sfa_kv_pages`` of an int32 table with unit column stride, which must
    outlive the call."""
    if (num_pages | block_table.shape[1] | page_size) >> 31:
        raise ValueError(f"a pool of {num_pages} pages of {page_size} rows or a table of {block_table.shape[1]} pages a sequence "
                         "is past 2^31")
    pg = _lib.KvPages()
    pg.block_table, pg.bt_sb = block_table.data_ptr(), block_table.stride(0)
    pg.max_pages, pg.page_size, pg.num_pages, pg.flags = block_table.shape[1], page_size, num_pages, 0
    return pg


def table(block_table: torch.Tensor, B: int, device: torch.device) -> torch.Tensor:
    """The block table as the kernels read it: int32, unit column stride."""
    need_gpu("block_table", block_table, device)
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.dtype not in INTS:
        raise ValueError(f"block_table must be an integer [B, max_pages] tensor with B = {B}, got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    bt = int32(block_table)
    if bt.stride(1) != 1 or (B > 1 and bt.stride(0) < bt.shape[1]):
        bt = bt.contiguous()
    return bt
