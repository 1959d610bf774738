"""Norm and rotation of the query and key heads, the step between the projections and the
attention, fused into one sm_100a pass (``ifa4_qk_norm_rope_launch``, include/inkling_fa4.h), its
gradients, and the same step with the append of keys and values to the paged cache
(``ifa4_kv_append_launch``).

The reference repository has these steps only in its diagram (outputs/architecture.md:18-64 and
:117-120).  Here, per token and head of 128 dims,

    y   = x * rsqrt(mean_i x_i^2 + eps) * w
    out = y with the pairs of its first ``2 * len(inv_freq)`` dims turned by pos * inv_freq[i]

in fp32 with one rounding to bf16; the pairs are ``(i, i + len(inv_freq))`` or, ``interleaved``,
``(2i, 2i + 1)``.  ``pos`` is the token's position in its sequence as the other entry points
count it: ``t - cu_seqlens_q[b]``, plus ``len_k - len_q`` when ``cu_seqlens_k`` is given.

The calls are no dispatcher operators: dispatch modes do not see them, and under ``make_fx`` or
``torch.jit.trace`` they are refused.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib, _ops

HEAD_DIM = _ops.HEAD_DIM
_NO_NORM = -1.0  # eps that the plain calls take for "no norm"


def _rows_ready(t: torch.Tensor) -> torch.Tensor:
    """Row tensors [tokens, heads, 128] are read in 16-byte pieces; anything else is copied."""
    st, sh, sd = t.stride()
    if sd == 1 and st % 8 == 0 and sh % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    return _ops.copy_rows(t)


def _eps(eps):
    """eps as the plain calls take it: -1 for no norm, NaN (never the plain case) for a value
    that the checks will refuse."""
    if eps is None:
        return _NO_NORM
    return eps if isinstance(eps, float) and 0 <= eps < math.inf else math.nan


def _empty_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _check_rows(name, nm, t, like, heads=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: {nm} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: {nm} must be a CUDA tensor (no CPU path exists)")
    if t.dtype is not torch.bfloat16:
        raise TypeError(f"{name}: {nm} must be bfloat16, got {t.dtype}")
    shape = t.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM:
        raise ValueError(f"{name}: {nm} must be [tokens, heads, {HEAD_DIM}], got {tuple(shape)}")
    if like is not None and (shape[0] != like.shape[0] or t.device != like.device):
        raise ValueError(f"{name}: {nm} must have the tokens and device of the other heads")
    if heads is not None and shape[1] != heads:
        raise ValueError(f"{name}: {nm} must have {heads} heads, got {shape[1]}")


def _check_written(name, nm, t):
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name}: {nm} needs unit last stride, strides multiple of 8, 16-B "
                         "alignment")


def _apart(a, b):
    """Whether the rows ``a`` and ``b`` [tokens, heads, 128] are known to have no element in common:
    they lie in different memory, one behind the other, or as columns of the same rows (slices of a
    merged projection) or heads in turn."""
    if (not a.numel() or not b.numel()
            or a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr()):
        return True

    def end(t):  # elements from the first to behind the last
        return sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1

    at = (b.data_ptr() - a.data_ptr()) // a.element_size()
    if at >= end(a) or -at >= end(b):
        return True

    def within(step, a_width, b_width):  # modulo step, [0, a_width) and [at, at + b_width) are apart
        return step > 0 and a_width <= at % step <= step - b_width

    (at_, ah, _), (bt, bh, _) = a.stride(), b.stride()
    return (at_ == bt and within(bt, end(a[0]), end(b[0]))
            or ah == bh and ah > 0 and at_ % ah == 0 and bt % ah == 0
            and within(ah, HEAD_DIM, HEAD_DIM))


def _check_cu(name, device, cu_q, cu_k):
    for nm, cu in (("cu_seqlens_q", cu_q), ("cu_seqlens_k", cu_k)):
        if cu is not None and (not isinstance(cu, torch.Tensor) or cu.dtype is not torch.int32
                               or cu.dim() != 1 or cu.numel() < 2 or cu.device != device):
            raise ValueError(f"{name}: {nm} must be a 1-D int32 tensor [batch + 1] on the inputs' "
                             "device")
    if cu_k is not None:
        if cu_q is None:
            raise ValueError(f"{name}: cu_seqlens_k needs cu_seqlens_q")
        if cu_k.numel() != cu_q.numel():
            raise ValueError(f"{name}: cu_seqlens_q and cu_seqlens_k differ in length")
    return (None if cu_q is None else cu_q.contiguous(),
            None if cu_k is None else cu_k.contiguous())


def _check_step(name, device, q_weight, k_weight, eps, inv_freq):
    """Weights, eps and frequencies; returns them as the operators take them."""
    dtype = None
    for nm, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if not isinstance(w, torch.Tensor) or w.device != device or w.shape != (HEAD_DIM,):
            raise ValueError(f"{name}: {nm} must be a [{HEAD_DIM}] tensor on the inputs' device")
        if w.dtype is not torch.bfloat16 and w.dtype is not torch.float32:
            raise TypeError(f"{name}: {nm} must be bfloat16 or float32, got {w.dtype}")
        if dtype is not None and w.dtype is not dtype:
            raise TypeError(f"{name}: q_weight and k_weight differ in dtype")
        dtype = w.dtype
    if eps is None:
        if dtype is not None:
            raise ValueError(f"{name}: weights without the norm (eps is None)")
        eps = _NO_NORM
    else:
        eps = float(eps)
        if not (eps >= 0 and math.isfinite(eps)):
            raise ValueError(f"{name}: eps must be finite and >= 0, or None for no norm")
    if inv_freq is not None:
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.device != device:
            raise ValueError(f"{name}: inv_freq must be a tensor on the inputs' device")
        if inv_freq.dtype is not torch.float64 and inv_freq.dtype is not torch.float32:
            raise TypeError(f"{name}: inv_freq must be float64 or float32, got {inv_freq.dtype}")
        n = inv_freq.numel()
        if inv_freq.dim() != 1 or n % 8 or not 0 < n <= HEAD_DIM // 2:
            raise ValueError(f"{name}: inv_freq must be 1-D with 8, 16, .., {HEAD_DIM // 2} "
                             f"entries, got {tuple(inv_freq.shape)}")
        inv_freq = inv_freq.contiguous()
    return (None if q_weight is None else q_weight.contiguous(),
            None if k_weight is None else k_weight.contiguous(), eps, inv_freq)


def _fill_step(p, heads, kv_heads, q_weight, k_weight, cu_q, cu_k, eps, inv_freq, interleaved,
               total_q):
    p.q_weight = None if q_weight is None else q_weight.data_ptr()
    p.k_weight = None if k_weight is None else k_weight.data_ptr()
    p.inv_freq = None if inv_freq is None else inv_freq.data_ptr()
    p.cu_seqlens_q = None if cu_q is None else cu_q.data_ptr()
    p.cu_seqlens_k = None if cu_k is None else cu_k.data_ptr()
    p.total_q = total_q
    p.batch = 1 if cu_q is None else cu_q.numel() - 1
    p.n_heads, p.kv_heads, p.head_dim = heads, kv_heads, HEAD_DIM
    p.rotary_dim = 0 if inv_freq is None else 2 * inv_freq.numel()
    p.interleaved = int(bool(interleaved))
    p.normalize = int(eps >= 0)
    w = q_weight if q_weight is not None else k_weight
    p.weight_dtype = _lib.IFA4_WEIGHT_F32 if w is not None and w.dtype is torch.float32 \
        else _lib.IFA4_WEIGHT_BF16
    p.inv_freq_f32 = int(inv_freq is not None and inv_freq.dtype is torch.float32)
    p.dtype = _lib.IFA4_DTYPE_BF16
    p.eps = max(eps, 0.0)


def _fill_rows(p, **tensors):
    for nm, t in tensors.items():
        setattr(p, nm, t.data_ptr())
        setattr(p, f"{nm}_stride_t", t.stride(0))
        setattr(p, f"{nm}_stride_h", t.stride(1))


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _forward(q, k, q_weight, k_weight, cu_q, cu_k, eps, inv_freq, interleaved):
    name = "qk_norm_rope"
    if _ops.USE_TORCH_OPS:
        outs = _lib.plain_call("qk_norm_rope", q, k, q_weight, k_weight, inv_freq, cu_q, cu_k,
                               interleaved, _eps(eps))
        if outs is not None:
            return outs[0], outs[1]
    _ops.refuse_tracing(name)
    _check_rows(name, "q", q, None)
    _check_rows(name, "k", k, q)
    cu_q, cu_k = _check_cu(name, q.device, cu_q, cu_k)
    q_weight, k_weight, eps, inv_freq = _check_step(name, q.device, q_weight, k_weight, eps,
                                                    inv_freq)
    if eps < 0 and inv_freq is None:
        raise ValueError(f"{name}: neither a norm (eps) nor a rotation (inv_freq)")
    q, k = _rows_ready(q), _rows_ready(k)
    q_out, k_out = _empty_like(q), _empty_like(k)
    p = _lib.QkNormRopeParams()
    _fill_rows(p, q=q, k=k, q_out=q_out, k_out=k_out)
    _fill_step(p, q.shape[1], k.shape[1], q_weight, k_weight, cu_q, cu_k, eps, inv_freq,
               interleaved, q.shape[0])
    p.zero_padding = 1
    with torch.cuda.device(q.device):
        _lib.check(_lib.lib().ifa4_qk_norm_rope_launch(ctypes.byref(p), _stream(q.device)))
    return q_out, k_out


def _backward(dq_out, dk_out, q, k, q_weight, k_weight, cu_q, cu_k, eps, inv_freq, interleaved,
              weight_grads):
    name = "qk_norm_rope_backward"
    if _ops.USE_TORCH_OPS:
        outs = _lib.plain_call("qk_norm_rope_backward", dq_out, dk_out, q, k, q_weight, k_weight,
                               inv_freq, cu_q, cu_k, interleaved, _eps(eps), *weight_grads)
        if outs is not None:
            dq, dk, *dw = outs
            dqw = dw.pop(0) if q_weight is not None and weight_grads[0] else None
            return dq, dk, dqw, dw.pop(0) if dw else None
    return _checked_backward(name, dq_out, dk_out, q, k, q_weight, k_weight, cu_q, cu_k, eps,
                             inv_freq, interleaved, weight_grads)


@torch.no_grad()
def _checked_backward(name, dq_out, dk_out, q, k, q_weight, k_weight, cu_q, cu_k, eps, inv_freq,
                      interleaved, weight_grads):
    _ops.refuse_tracing(name)
    _check_rows(name, "q", q, None)
    _check_rows(name, "k", k, q)
    _check_rows(name, "dq_out", dq_out, q, q.shape[1])
    _check_rows(name, "dk_out", dk_out, q, k.shape[1])
    cu_q, cu_k = _check_cu(name, q.device, cu_q, cu_k)
    q_weight, k_weight, eps, inv_freq = _check_step(name, q.device, q_weight, k_weight, eps,
                                                    inv_freq)
    q, k, dq_out, dk_out = (_rows_ready(t) for t in (q, k, dq_out, dk_out))
    dq, dk = _empty_like(q), _empty_like(k)
    dqw = torch.empty_like(q_weight) if q_weight is not None and weight_grads[0] else None
    dkw = torch.empty_like(k_weight) if k_weight is not None and weight_grads[1] else None
    p = _lib.QkNormRopeBackwardParams()
    _fill_rows(p, dq_out=dq_out, dk_out=dk_out, q=q, k=k, dq=dq, dk=dk)
    _fill_step(p, q.shape[1], k.shape[1], q_weight, k_weight, cu_q, cu_k, eps, inv_freq,
               interleaved, q.shape[0])
    p.dq_weight = None if dqw is None else dqw.data_ptr()
    p.dk_weight = None if dkw is None else dkw.data_ptr()
    L = _lib.lib()
    with torch.cuda.device(q.device):
        need = ctypes.c_size_t(0)
        _lib.check(L.ifa4_qk_norm_rope_backward_workspace_size(ctypes.byref(p), ctypes.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
        _lib.check(L.ifa4_qk_norm_rope_backward_launch(
            ctypes.byref(p), ctypes.c_void_p(0 if ws is None else ws.data_ptr()), need,
            _stream(q.device)))
    return dq, dk, dqw, dkw


class QkNormRopeFunction(torch.autograd.Function):
    """Saves the inputs only; the backward recomputes the norms."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cu_q, cu_k, eps, inv_freq, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, cu_q, cu_k, inv_freq)
        ctx.step = (eps, interleaved)
        return _forward(q, k, q_weight, k_weight, cu_q, cu_k, eps, inv_freq, interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cu_q, cu_k, inv_freq = ctx.saved_tensors
        eps, interleaved = ctx.step
        dq, dk, dqw, dkw = _backward(dq_out, dk_out, q, k, q_weight, k_weight, cu_q, cu_k, eps,
                                     inv_freq, interleaved, ctx.needs_input_grad[2:4])
        return dq, dk, dqw, dkw, None, None, None, None, None


def inkling_qk_norm_rope(q, k, q_weight=None, k_weight=None, cu_seqlens_q=None, cu_seqlens_k=None,
                         *, eps=1e-6, inv_freq=None, interleaved=False):
    """Normalised and rotated ``(q_out, k_out)`` of ``q [total_q, n_heads, 128]`` and
    ``k [total_q, kv_heads, 128]`` (bf16; slices of a merged projection are read in place),
    differentiable in q, k and the weights (once, and not in forward mode, which is refused).

    ``q_weight`` / ``k_weight``: ``[128]`` bf16 or fp32 (None: ones).  ``eps=None``: no norm.
    ``inv_freq``: ``[rotary_dim / 2]`` fp64 or fp32 tensor of angles per position, 8, 16, .., 64
    entries (None: no rotation); angles are good to 64-bit arithmetic, 1e-6 rad at position 2^31.
    ``interleaved`` pairs neighbouring dims instead of the two halves.  Rows behind the last sequence
    (``cu_seqlens_q[batch]``) come out as zeros, and so do their gradients, which count in no
    weight gradient."""
    if _ops.differentiates(q, k, q_weight, k_weight):
        return QkNormRopeFunction.apply(q, k, q_weight, k_weight, cu_seqlens_q, cu_seqlens_k, eps,
                                        inv_freq, interleaved)
    return _forward(q, k, q_weight, k_weight, cu_seqlens_q, cu_seqlens_k, eps, inv_freq,
                    interleaved)


def inkling_qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight=None, k_weight=None,
                                  cu_seqlens_q=None, cu_seqlens_k=None, *, eps=1e-6,
                                  inv_freq=None, interleaved=False):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of ``inkling_qk_norm_rope`` given those of its
    outputs; a weight that is None has the gradient None.  Sums are fp32 in a fixed order (the
    same result every time)."""
    return _backward(dq_out, dk_out, q, k, q_weight, k_weight, cu_seqlens_q, cu_seqlens_k, eps,
                     inv_freq, interleaved, (True, True))


def inkling_kv_append(k, v, k_cache, v_cache, block_table, cu_seqlens_q, cu_seqlens_k, *, q=None,
                      q_weight=None, k_weight=None, eps=1e-6, inv_freq=None, interleaved=False,
                      q_out=None):
    """Appends new tokens to a paged cache, normalising and rotating the keys on the way, and
    optionally does the same for their queries in the same launch.

    ``k, v [total_q, kv_heads, 128]`` are the new tokens of all sequences (rows
    ``cu_seqlens_q[b] .. cu_seqlens_q[b + 1]``), which are the last of the sequence's
    ``cu_seqlens_k[b + 1] - cu_seqlens_k[b]`` keys: the key counts include them, as the
    attention call that follows takes them.  The token at position ``p`` goes to page
    ``block_table[b, p // page_size]``, slot ``p % page_size`` of ``k_cache`` and ``v_cache
    [num_pages, page_size, kv_heads, 128]`` (page_size a power of two >= 16).  ``v`` is copied;
    ``k`` and ``q`` take the step of ``inkling_qk_norm_rope`` (``eps=None`` and no ``inv_freq``:
    copied too).  A token without a place (a table entry outside ``[0, num_pages)``, a position
    below 0 or past the table, a row behind the last sequence) writes nothing to the caches.
    No two tokens of a call may have the same place, and ``k``, ``v`` and ``q`` must not lie in places
    that the call writes.

    Not differentiable: the queries that come back are cut off from ``q``'s graph, and a backward
    that saved a cache (or ``q``, where ``q_out`` is ``q``) from before the call raises.

    Returns the queries (``q_out`` if given, which may be ``q`` itself, where ``k`` and ``v`` have no
    element in common with it: rows behind the last sequence are then left as they were; a new
    tensor has zeros there), or None without ``q``."""
    if q is not None and q_out is None and _ops.USE_TORCH_OPS:
        outs = _lib.plain_call("kv_append", q, k, v, k_cache, v_cache, q_weight, k_weight,
                               inv_freq, cu_seqlens_q, cu_seqlens_k, block_table, interleaved,
                               _eps(eps))
        if outs is not None:
            return outs[0]
    return _checked_append(k, v, k_cache, v_cache, block_table, cu_seqlens_q, cu_seqlens_k, q,
                           q_weight, k_weight, eps, inv_freq, interleaved, q_out)


@torch.no_grad()
def _checked_append(k, v, k_cache, v_cache, block_table, cu_seqlens_q, cu_seqlens_k, q, q_weight,
                    k_weight, eps, inv_freq, interleaved, q_out):
    name = "kv_append"
    _ops.refuse_tracing(name)
    _check_rows(name, "k", k, None)
    _check_rows(name, "v", v, k, k.shape[1])
    device = k.device
    if cu_seqlens_q is None or cu_seqlens_k is None:
        raise ValueError(f"{name}: needs cu_seqlens_q and cu_seqlens_k")
    cu_seqlens_q, cu_seqlens_k = _check_cu(name, device, cu_seqlens_q, cu_seqlens_k)
    q_weight, k_weight, eps, inv_freq = _check_step(name, device, q_weight, k_weight, eps,
                                                    inv_freq)
    for nm, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: {nm} must be a torch.Tensor")
        if t.dtype is not torch.bfloat16:
            raise TypeError(f"{name}: {nm} must be bfloat16, got {t.dtype}")
        if t.device != device or t.dim() != 4 or t.shape[2] != k.shape[1] or t.shape[3] != HEAD_DIM:
            raise ValueError(f"{name}: {nm} must be [num_pages, page_size, kv_heads, {HEAD_DIM}] "
                             "on k's device")
        if not _ops.tma_layout(t):
            raise ValueError(f"{name}: {nm} needs unit last stride, strides that are positive "
                             "multiples of 8 elements, 16-byte alignment")
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"{name}: k_cache and v_cache differ in shape")
    if k_cache.data_ptr() == v_cache.data_ptr() and k_cache.numel():
        raise ValueError(f"{name}: k_cache and v_cache are the same memory")
    page_size = k_cache.shape[1]
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"{name}: page_size {page_size} must be a power of two >= 16")
    if (not isinstance(block_table, torch.Tensor) or block_table.device != device
            or block_table.dtype is not torch.int32 or block_table.dim() != 2
            or block_table.shape[0] != cu_seqlens_q.numel() - 1):
        raise ValueError(f"{name}: block_table must be int32 [batch, max_pages] on k's device")
    block_table = _ops._table(block_table)
    k, v = _rows_ready(k), _rows_ready(v)
    zero_padding = q_out is None
    if q is None:
        if q_out is not None or q_weight is not None:
            raise ValueError(f"{name}: q_out or q_weight without q")
    else:
        _check_rows(name, "q", q, k)
        if q_out is None:
            q = _rows_ready(q)
            q_out = _empty_like(q)
        else:
            _check_rows(name, "q_out", q_out, k, q.shape[1])
            _check_written(name, "q_out", q_out)
            same = q_out.data_ptr() == q.data_ptr() and q_out.stride() == q.stride()
            store = q_out.untyped_storage().data_ptr()
            if not same and any(t.untyped_storage().data_ptr() == store for t in (q, k, v)):
                raise ValueError(f"{name}: q_out must be q itself or share no storage with q, k, v")
            if not (_apart(q_out, k) and _apart(q_out, v)):
                raise ValueError(f"{name}: k and v must have no element in common with q_out")
            q = _rows_ready(q)
    p = _lib.KvAppendParams()
    _fill_rows(p, k=k, v=v)
    if q is not None:
        _fill_rows(p, q=q, q_out=q_out)
    _fill_step(p, 0 if q is None else q.shape[1], k.shape[1], q_weight, k_weight, cu_seqlens_q,
               cu_seqlens_k, eps, inv_freq, interleaved, k.shape[0])
    p.zero_padding = int(zero_padding)
    p.k_cache, p.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    p.k_stride_page, p.k_cache_stride_t, p.k_cache_stride_h = k_cache.stride()[:3]
    p.v_stride_page, p.v_cache_stride_t, p.v_cache_stride_h = v_cache.stride()[:3]
    p.block_table, p.block_table_stride = block_table.data_ptr(), block_table.stride(0)
    p.page_size, p.num_pages = page_size, k_cache.shape[0]
    p.table_width = block_table.shape[1]
    with torch.cuda.device(device):
        _lib.check(_lib.lib().ifa4_kv_append_launch(ctypes.byref(p), _stream(device)))
    _ops.written(k_cache, v_cache, None if zero_padding else q_out)
    return q_out


__all__ = ["inkling_qk_norm_rope", "inkling_qk_norm_rope_backward", "inkling_kv_append",
           "QkNormRopeFunction"]
