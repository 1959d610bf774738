"""Checks and parameter blocks that the long-context operators over the paged cache share
(``page_sparse``, ``kv_evict``)."""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib, _ops

HEAD_DIM = _ops.HEAD_DIM
MOST = 1 << 26  # entries of a table row or of a choice
MOST_DISTANCES = 1 << 29


def tensor(name, nm, t, device, dtype, dims):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: {nm} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: {nm} must be a CUDA tensor (no CPU path exists)")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: {nm} is on {t.device}, the other tensors on {device}")
    if t.dtype is not dtype:
        raise TypeError(f"{name}: {nm} must be {dtype}, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name}: {nm} must have {dims} dimensions, got {tuple(t.shape)}")


def cache(name, nm, t, device=None):
    """A paged cache ``[num_pages, page_size, kv_heads, 128]``, never copied."""
    tensor(name, nm, t, device, torch.bfloat16, 4)
    if t.shape[3] != HEAD_DIM or t.shape[2] < 1:
        raise ValueError(f"{name}: {nm} must be [num_pages, page_size, kv_heads, {HEAD_DIM}], got "
                         f"{tuple(t.shape)}")
    page_size(name, t.shape[1])
    _in_place(name, nm, t)


def _in_place(name, nm, t):
    if t.numel() and not _ops.tma_layout(t):
        raise ValueError(f"{name}: {nm} needs unit last stride, strides that are positive multiples "
                         "of 8 elements, 16-byte alignment")


def page_size(name, n):
    if type(n) is not int or n < 16 or n > 1 << 20 or n & (n - 1):
        raise ValueError(f"{name}: page_size {n} must be a power of two in [16, 2^20]")


def page_bounds(name, t, kv_heads, num_pages, device):
    tensor(name, "bounds", t, device, torch.bfloat16, 4)
    if t.shape[2:] != (2, HEAD_DIM) or (kv_heads is not None and t.shape[1] != kv_heads) or (
            num_pages is not None and t.shape[0] != num_pages):
        raise ValueError(f"{name}: bounds must be [num_pages, kv_heads, 2, {HEAD_DIM}] of the cache's "
                         f"pages and heads, got {tuple(t.shape)}")
    _in_place(name, "bounds", t)
    if t.numel() and t.stride(2) != HEAD_DIM:
        raise ValueError(f"{name}: minima and maxima of a page and head must be contiguous in bounds")


def distances(name, rel_extent):
    if rel_extent > MOST_DISTANCES:
        raise ValueError(f"{name}: rel_extent {rel_extent} must be at most 2^29")


def sequences(name, device, cu_q, cu_k, block_table):
    """Checked offsets and table as the kernels read them."""
    for nm, cu in (("cu_seqlens_q", cu_q), ("cu_seqlens_k", cu_k)):
        tensor(name, nm, cu, device, torch.int32, 1)
        if cu.numel() < 2:
            raise ValueError(f"{name}: {nm} must be [batch + 1] with a sequence at least")
    if cu_q.numel() != cu_k.numel():
        raise ValueError(f"{name}: cu_seqlens_q and cu_seqlens_k differ in length")
    tensor(name, "block_table", block_table, device, torch.int32, 2)
    if block_table.shape[0] != cu_q.numel() - 1 or block_table.shape[1] > MOST:
        raise ValueError(f"{name}: block_table must be [batch, max_pages], at most 2^26 pages wide")
    return _ops._offsets(cu_q), _ops._offsets(cu_k), _ops._table(block_table)


def queries(name, q, rel_logits, kv_heads, rel_extent, softmax_scale, device):
    """Checked queries and bias as the kernels read them, the extent and the scale."""
    tensor(name, "q", q, device, torch.bfloat16, 3)
    tensor(name, "rel_logits", rel_logits, device, torch.bfloat16, 3)
    if q.shape[2] != HEAD_DIM or q.shape[1] < 1 or q.shape[1] % kv_heads:
        raise ValueError(f"{name}: q must be [total_q, n_heads, {HEAD_DIM}] with n_heads a multiple of "
                         f"kv_heads {kv_heads}, got {tuple(q.shape)}")
    if rel_logits.shape[:2] != q.shape[:2]:
        raise ValueError(f"{name}: rel_logits must be [total_q, n_heads, >=rel_extent]")
    rel_extent = int(rel_extent)
    if rel_extent <= 0 or rel_logits.shape[2] < rel_extent:
        raise ValueError(f"{name}: rel_extent {rel_extent} out of range for rel_logits "
                         f"{tuple(rel_logits.shape)}")
    distances(name, rel_extent)
    scale = 1.0 / HEAD_DIM if softmax_scale is None else float(softmax_scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{name}: softmax_scale must be > 0")
    rel = rel_logits if rel_logits.stride(-1) == 1 else rel_logits.contiguous()
    return _ops._tma_ready(q) if q.numel() else q, rel, rel_extent, scale


def rows_apart(t):
    """Unit last stride, and no two rows of the first two dimensions share an element."""
    if t.shape[2] > 1 and t.stride(2) != 1:
        return False
    rows = sorted((t.stride(i), t.shape[i]) for i in (0, 1) if t.shape[i] > 1)
    reach = t.shape[2]  # elements that the rows so far take up
    for stride, count in rows:
        if stride < reach:
            return False
        reach += stride * (count - 1)
    return True


def hint(n):
    """A length that sizes the grid (0: not known)."""
    return min(max(int(n), 0), 0x7fffffff) if n else 0


def window(window_size):
    return min(int(window_size[0]), 0x7fffffff) if window_size is not None else -1


def fill_seqs(p, cu_q, cu_k, block_table, size, num_pages):
    s = p.seqs
    s.cu_seqlens_q, s.cu_seqlens_k = cu_q.data_ptr(), cu_k.data_ptr()
    s.block_table, s.block_table_stride = block_table.data_ptr(), block_table.stride(0)
    s.batch, s.table_width = cu_q.numel() - 1, block_table.shape[1]
    s.page_size, s.num_pages = size, num_pages


def fill_strides(p, **tensors):
    """``<name>_stride_<suffix>`` of every tensor, suffixes in the order of its dimensions."""
    for nm, (t, suffixes) in tensors.items():
        for suffix, stride in zip(suffixes, t.stride()):
            setattr(p, f"{nm}_stride_{suffix}", stride)


def launch(entry, p, device, workspace=None, sized=False):
    """Launches on the device's current stream; with ``sized`` the entry point takes a workspace,
    allocated here where the given one is absent or too small."""
    L = _lib.lib()
    with torch.cuda.device(device):
        stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
        call = getattr(L, f"ifa4_{entry}_launch")
        if not sized:
            _lib.check(call(ctypes.byref(p), stream))
            return
        need = ctypes.c_size_t(0)
        _lib.check(getattr(L, f"ifa4_{entry}_workspace_size")(ctypes.byref(p), ctypes.byref(need)))
        if need.value and (workspace is None
                           or workspace.numel() * workspace.element_size() < need.value):
            workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        ptr = workspace.data_ptr() if need.value else 0
        _lib.check(call(ctypes.byref(p), ctypes.c_void_p(ptr), need, stream))
