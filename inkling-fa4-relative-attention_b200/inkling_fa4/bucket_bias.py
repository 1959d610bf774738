"""Learned relative position bias by distance buckets: the other source of the attention's
``rel_logits`` next to ``inkling_rel_logits``, with its gradient (``ifa4_bucket_bias_launch`` and
``ifa4_bucket_bias_backward_launch``, include/inkling_fa4.h).

A table holds one value per bucket and head; ``rel_logits[t, h, d] = table[bucket(d), h]`` for the
distances ``0 <= d < rel_extent``, where ``bucket(d)`` is the last bucket whose start is <= d.  It
is the same for every token, so the result is one ``[n_heads, rel_extent]`` table seen through
token stride 0, which the attention entry points read as it is.  The gradient adds the
attention's d rel_logits over tokens and over each bucket's distances.

The calls are no dispatcher operators: dispatch modes do not see them, and under ``make_fx`` or
``torch.jit.trace`` they are refused."""
from __future__ import annotations

import ctypes

import torch

from . import _lib, _ops


def relative_bucket_starts(num_buckets: int, max_distance: int) -> list:
    """First distance of each of ``num_buckets`` buckets: half of them hold one distance each, the
    others grow logarithmically up to ``max_distance``, the last one taking all distances beyond
    (with ``e = num_buckets // 2`` and ``n = num_buckets - e``, bucket ``e + j`` starts at the first
    distance d with ``(d / e)^n >= (max_distance / e)^j``, decided in whole numbers)."""
    num_buckets, max_distance = int(num_buckets), int(max_distance)
    if not 2 <= num_buckets <= _lib.MAX_BUCKETS:
        raise ValueError(f"relative_bucket_starts: num_buckets must be in [2, {_lib.MAX_BUCKETS}]")
    if max_distance < num_buckets:
        raise ValueError("relative_bucket_starts: max_distance must be >= num_buckets")
    e = num_buckets // 2
    n = num_buckets - e
    starts, d = list(range(e)), e
    for j in range(n):
        want = max_distance ** j * e ** (n - j)
        lo, hi = d, max_distance  # d^n >= want holds at max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            if mid ** n >= want:
                hi = mid
            else:
                lo = mid + 1
        d = lo
        starts.append(d)
    return starts


def _check_starts(name, starts, device):
    if (not isinstance(starts, torch.Tensor) or starts.dtype is not torch.int32
            or starts.dim() != 1 or starts.device != device):
        raise ValueError(f"{name}: starts must be a 1-D int32 tensor on the inputs' device")
    if not 1 <= starts.numel() <= _lib.MAX_BUCKETS:
        raise ValueError(f"{name}: 1 to {_lib.MAX_BUCKETS} buckets, got {starts.numel()}")
    return starts.contiguous()


def _weight_dtype(name, dtype):
    if dtype is torch.float32:
        return _lib.IFA4_WEIGHT_F32
    if dtype is torch.bfloat16:
        return _lib.IFA4_WEIGHT_BF16
    raise TypeError(f"{name}: the table must be bfloat16 or float32, got {dtype}")


def _forward(table, starts, total_q, rel_extent):
    name = "bucket_bias"
    if _ops.USE_TORCH_OPS:
        outs = _lib.plain_call("bucket_bias", table, starts, total_q, rel_extent)
        if outs is not None:
            return outs[0]
    _ops.refuse_tracing(name)
    if not isinstance(table, torch.Tensor):
        raise TypeError(f"{name}: table must be a torch.Tensor")
    if not table.is_cuda:
        raise ValueError(f"{name}: table must be a CUDA tensor (no CPU path exists)")
    wt = _weight_dtype(name, table.dtype)
    starts = _check_starts(name, starts, table.device)
    if table.dim() != 2 or table.shape[0] != starts.numel() or table.shape[1] < 1:
        raise ValueError(f"{name}: table must be [{starts.numel()} buckets, n_heads], got "
                         f"{tuple(table.shape)}")
    total_q, rel_extent = int(total_q), int(rel_extent)
    if total_q < 0 or not 0 < rel_extent <= 1 << 24:
        raise ValueError(f"{name}: total_q must be >= 0, rel_extent in [1, 2^24]")
    heads = table.shape[1]
    rel = torch.empty((heads, rel_extent), dtype=torch.bfloat16, device=table.device)
    p = _lib.BucketBiasParams()
    p.table, p.starts, p.rel = table.data_ptr(), starts.data_ptr(), rel.data_ptr()
    p.table_stride_b, p.table_stride_h = table.stride()
    p.rel_stride_h = rel_extent
    p.n_heads, p.rel_extent, p.buckets, p.weight_dtype = heads, rel_extent, starts.numel(), wt
    with torch.cuda.device(table.device):
        stream = torch.cuda.current_stream(table.device).cuda_stream
        _lib.check(_lib.lib().ifa4_bucket_bias_launch(ctypes.byref(p), ctypes.c_void_p(stream)))
    return rel.unsqueeze(0).expand(total_q, heads, rel_extent)


def _backward(drel, starts, dtype, cu_seqlens_q):
    if _ops.USE_TORCH_OPS and (dtype is torch.float32 or dtype is torch.bfloat16):
        outs = _lib.plain_call("bucket_bias_backward", drel, starts, dtype is torch.float32,
                               cu_seqlens_q)
        if outs is not None:
            return outs[0]
    return _checked_backward(drel, starts, dtype, cu_seqlens_q)


@torch.no_grad()
def _checked_backward(drel, starts, dtype, cu_seqlens_q):
    name = "bucket_bias_backward"
    _ops.refuse_tracing(name)
    if not isinstance(drel, torch.Tensor):
        raise TypeError(f"{name}: drel must be a torch.Tensor")
    if not drel.is_cuda:
        raise ValueError(f"{name}: drel must be a CUDA tensor (no CPU path exists)")
    if drel.dtype is not torch.bfloat16:
        raise TypeError(f"{name}: drel must be bfloat16, got {drel.dtype}")
    if drel.dim() != 3 or drel.shape[1] < 1 or not 0 < drel.shape[2] <= 1 << 24:
        raise ValueError(f"{name}: drel must be [total_q, n_heads, rel_extent], got "
                         f"{tuple(drel.shape)}")
    starts = _check_starts(name, starts, drel.device)
    wt = _weight_dtype(name, dtype)
    if cu_seqlens_q is not None:
        if (not isinstance(cu_seqlens_q, torch.Tensor) or cu_seqlens_q.dtype is not torch.int32
                or cu_seqlens_q.dim() != 1 or cu_seqlens_q.numel() < 1
                or cu_seqlens_q.device != drel.device):
            raise ValueError(f"{name}: cu_seqlens_q must be a 1-D int32 tensor [batch + 1] on "
                             "drel's device")
        cu_seqlens_q = cu_seqlens_q.contiguous()
    if drel.stride(2) != 1 and drel.shape[2] > 1:
        drel = drel.contiguous()
    heads, buckets = drel.shape[1], starts.numel()
    dtable = torch.empty((buckets, heads), dtype=dtype, device=drel.device)
    p = _lib.BucketBiasBackwardParams()
    p.drel, p.starts, p.dtable = drel.data_ptr(), starts.data_ptr(), dtable.data_ptr()
    p.cu_seqlens_q = None if cu_seqlens_q is None else cu_seqlens_q.data_ptr()
    p.drel_stride_t, p.drel_stride_h = drel.stride()[:2]
    p.dtable_stride_b, p.dtable_stride_h = dtable.stride()
    p.total_q = drel.shape[0]
    p.batch = 0 if cu_seqlens_q is None else cu_seqlens_q.numel() - 1
    p.n_heads, p.rel_extent, p.buckets, p.weight_dtype = heads, drel.shape[2], buckets, wt
    L = _lib.lib()
    with torch.cuda.device(drel.device):
        need = ctypes.c_size_t(0)
        _lib.check(L.ifa4_bucket_bias_backward_workspace_size(ctypes.byref(p), ctypes.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=drel.device) if need.value else None
        stream = torch.cuda.current_stream(drel.device).cuda_stream
        _lib.check(L.ifa4_bucket_bias_backward_launch(
            ctypes.byref(p), ctypes.c_void_p(0 if ws is None else ws.data_ptr()), need,
            ctypes.c_void_p(stream)))
    return dtable


class BucketBiasFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, starts, total_q, rel_extent, cu_seqlens_q):
        ctx.save_for_backward(starts, cu_seqlens_q)
        ctx.dtype = table.dtype
        return _forward(table, starts, total_q, rel_extent)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drel):
        starts, cu_seqlens_q = ctx.saved_tensors
        return _backward(drel, starts, ctx.dtype, cu_seqlens_q), None, None, None, None


def inkling_bucket_bias(table, starts, total_q, rel_extent, cu_seqlens_q=None):
    """``rel_logits [total_q, n_heads, rel_extent]`` (bf16, token stride 0) of a learned ``table
    [num_buckets, n_heads]`` (bf16 or fp32) whose buckets begin at the distances ``starts
    [num_buckets]`` (int32 on the device, ascending; ``relative_bucket_starts`` makes the usual
    ones).  Differentiable in ``table`` (once, and not in forward mode, which is refused); the
    gradient counts the tokens before ``cu_seqlens_q[-1]`` (None: all).  The result is a view for
    reading: its tokens are the same memory."""
    if _ops.differentiates(table):
        return BucketBiasFunction.apply(table, starts, total_q, rel_extent, cu_seqlens_q)
    return _forward(table, starts, total_q, rel_extent)


def inkling_bucket_bias_backward(drel, starts, num_buckets, *, dtype=torch.float32,
                                 cu_seqlens_q=None):
    """Gradient ``[num_buckets, n_heads]`` (``dtype`` float32 or bfloat16) of the table given the
    attention's ``drel [total_q, n_heads, rel_extent]`` (bf16): fp32 sums over the tokens before
    ``cu_seqlens_q[-1]`` (None: all) and each bucket's distances, in a fixed order (the same result
    every time)."""
    if isinstance(starts, torch.Tensor) and starts.numel() != int(num_buckets):
        raise ValueError(f"bucket_bias_backward: {starts.numel()} starts for {num_buckets} buckets")
    return _backward(drel, starts, dtype, cu_seqlens_q)


__all__ = ["inkling_bucket_bias", "inkling_bucket_bias_backward", "relative_bucket_starts",
           "BucketBiasFunction"]
