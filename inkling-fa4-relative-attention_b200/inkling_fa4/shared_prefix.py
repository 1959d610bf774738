"""Decode for a batch whose sequences begin with the same keys (a system prompt, a document that
several questions are asked about), which the plain decode would read once per sequence.  The call is
no dispatcher operator: dispatch modes do not see it, and under ``make_fx`` or ``torch.jit.trace`` it is
refused."""
from __future__ import annotations

import ctypes

import torch

from . import _lib, _ops


def inkling_fa4_rel_attention_decode_shared_prefix(q, k, v, rel_logits, cu_seqlens_q, cu_seqlens_k,
                                                   max_seqlen_q, max_seqlen_k, rel_extent,
                                                   shared_prefix_len, window_size=(-1, -1),
                                                   n_heads=None, kv_heads=None, head_dim=128, *,
                                                   block_table, softmax_scale=None, out=None,
                                                   prefix_splits=0, num_splits=0, chunk_len=0,
                                                   workspace=None, return_lse=False, lse=None):
    """The result of ``inkling_fa4_rel_attention_decode_triton(..., causal_align="bottom_right",
    block_table=block_table)`` on the same arguments, with the keys and values of positions
    ``[0, shared_prefix_len)`` read once for the batch: their part runs as a matrix product of
    all sequences' queries (tcgen05), the sequences' own keys through the decode kernel, and a
    merge combines the two.

    ``cu_seqlens_k`` counts all keys of a sequence, prefix included, and ``block_table`` rows
    list all its pages.  Every sequence of at least ``shared_prefix_len`` keys must hold the same
    keys and values there, as far as its window reaches; normally the table rows begin with the
    same pages, and the pages of one of these sequences, of those that are worked on together the
    one whose window reaches furthest back, are the ones that are read.  (A value among them that
    is no number reaches every sequence that is worked on with one that sees it.)  Sequences with
    fewer keys share nothing and are attended through their own pages; the automatic plan expects them
    to be short (a CTA per KV head walks all keys of one: a sequence of 30000 beside 16 behind 32k
    takes 293 us, 51 without it; give ``num_splits``, 92 us with 16, where there are such sequences).
    A logit that is no number, or +inf, makes its row NaN (the plain decode, and with it a prefix of
    0, leaves the keys that it was added up with out of the row).  ``shared_prefix_len`` is a host
    integer (it sizes the grid, at most 2^30) and need not be a multiple of the page size; 0 is a
    plain decode.

    One query per sequence (``cu_seqlens_q`` = 0..batch), at most 128 query heads per KV head.
    ``prefix_splits``: CTAs that share a row tile's prefix keys (0: automatic); ``num_splits`` /
    ``chunk_len``: the plan of the own keys, as in the decode.  ``workspace``: a reusable uint8
    CUDA tensor (allocated per call when absent or too small); calls that may run at the same
    time need one each."""
    if (out is None and lse is None and not return_lse and n_heads is None and kv_heads is None
            and head_dim == _ops.HEAD_DIM and _ops.USE_TORCH_OPS):
        outs = _lib.plain_call("decode_shared_prefix", q, k, v, rel_logits, cu_seqlens_q,
                               cu_seqlens_k, block_table, workspace, rel_extent,
                               -1 if window_size is None else window_size[0], max_seqlen_k or 0,
                               1.0 / _ops.HEAD_DIM if softmax_scale is None else softmax_scale,
                               num_splits, chunk_len, shared_prefix_len, prefix_splits)
        if outs is not None:
            return outs[0]
    return _checked(q, k, v, rel_logits, cu_seqlens_q, cu_seqlens_k, max_seqlen_k, rel_extent,
                    shared_prefix_len, window_size, n_heads, kv_heads, head_dim, block_table,
                    softmax_scale, out, prefix_splits, num_splits, chunk_len, workspace,
                    return_lse, lse)


@torch.no_grad()
def _checked(q, k, v, rel_logits, cu_seqlens_q, cu_seqlens_k, max_seqlen_k, rel_extent,
             shared_prefix_len, window_size, n_heads, kv_heads, head_dim, block_table,
             softmax_scale, out, prefix_splits, num_splits, chunk_len, workspace, return_lse, lse):
    given = (out, lse)
    name = "decode_shared_prefix"
    _ops.refuse_tracing(name)
    if block_table is None:
        raise ValueError(f"{name}: needs a paged cache (block_table)")
    block_table = _ops._table(block_table)
    cu_seqlens_q, cu_seqlens_k = _ops._offsets(cu_seqlens_q), _ops._offsets(cu_seqlens_k)
    q, k, v, rel, out, n_heads, kv_heads, rel_extent, window_left, scale = _ops._prepare(
        name, q, k, v, rel_logits, cu_seqlens_q, cu_seqlens_k, rel_extent, True, window_size,
        n_heads, kv_heads, head_dim, softmax_scale, "bottom_right", out, block_table)
    lse = _ops._lse_buffer(q, n_heads, return_lse, lse)
    if q.shape[0] != cu_seqlens_q.numel() - 1:
        raise ValueError(f"{name}: expects exactly one query token per sequence")
    shared_prefix_len = int(shared_prefix_len)
    if not 0 <= shared_prefix_len <= 1 << 30:
        raise ValueError(f"{name}: shared_prefix_len must be in [0, 2^30]")
    if shared_prefix_len > block_table.shape[1] * k.shape[1]:
        raise ValueError(f"{name}: shared_prefix_len {shared_prefix_len} is beyond the table's "
                         f"{block_table.shape[1]} pages of {k.shape[1]}")
    if workspace is not None and not (isinstance(workspace, torch.Tensor)
                                      and workspace.device == q.device
                                      and workspace.is_contiguous()):
        raise ValueError(f"{name}: workspace must be a contiguous tensor on q's device")
    max_seqlen_k = int(max_seqlen_k) if max_seqlen_k else 0
    p = _lib.SharedPrefixParams()
    p.decode = _ops._decode_params(q, k, v, rel, out, cu_seqlens_q, cu_seqlens_k, n_heads,
                                   kv_heads, rel_extent, True, window_left, "bottom_right",
                                   max_seqlen_k, scale, num_splits, chunk_len, block_table)
    _ops._fill_lse(p.decode, lse)
    p.shared_prefix_len, p.prefix_splits = shared_prefix_len, int(prefix_splits)
    L = _lib.lib()
    with torch.cuda.device(q.device):
        need = ctypes.c_size_t(0)
        _lib.check(L.ifa4_decode_shared_prefix_workspace_size(ctypes.byref(p), ctypes.byref(need)))
        if need.value and (workspace is None
                           or workspace.numel() * workspace.element_size() < need.value):
            workspace = torch.empty(need.value, dtype=torch.uint8, device=q.device)
        ptr = workspace.data_ptr() if need.value else 0
        stream = torch.cuda.current_stream(q.device).cuda_stream
        _lib.check(L.ifa4_decode_shared_prefix_launch(ctypes.byref(p), ctypes.c_void_p(ptr), need,
                                                      ctypes.c_void_p(stream)))
    _ops.written(*given)
    return (out, lse) if lse is not None else out


__all__ = ["inkling_fa4_rel_attention_decode_shared_prefix"]
