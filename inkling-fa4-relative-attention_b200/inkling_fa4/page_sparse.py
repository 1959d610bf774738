"""Sparse attention over the pages of a paged cache, for contexts of which a query needs a few pages
only: bounds of each page's keys, kept beside the cache; scores that bound the page's logits,
relative bias included; the choice of the highest; and attention over the chosen pages.  One layer's
step, behind the append::

    inkling_kv_page_bounds(k_cache, block_table, cu_q, cu_k, max_q, bounds=bounds)
    scores = inkling_kv_page_scores(q, bounds, rel, cu_q, cu_k, max_q, R, page_size,
                                    block_table=block_table, first_pages=1, last_pages=2)
    pages = inkling_kv_select_pages(scores, 64)
    out = inkling_fa4_rel_attention_decode_pages(q, k_cache, v_cache, rel, cu_q, cu_k, max_q, max_k, R,
                                                 pages, block_table=block_table)

Queries are the last of their sequence's keys (``causal_align="bottom_right"``), any number of them a
sequence, each with a choice of its own for every KV head.  The calls are no dispatcher operators and
not differentiable: what they return is cut off from the graph of their inputs; under ``make_fx`` and
``torch.jit.trace`` they are refused."""
from __future__ import annotations

import math

import torch

from . import _lib, _ops, _paged


def inkling_kv_page_bounds(k_cache, block_table, cu_seqlens_q, cu_seqlens_k, max_seqlen_q=None, *,
                           bounds=None):
    """Elementwise minimum and maximum of the keys of every page that holds one of the last
    ``cu_seqlens_q[b + 1] - cu_seqlens_q[b]`` tokens of a sequence, so the call behind an append
    takes the append's offsets; with ``cu_seqlens_q = cu_seqlens_k`` all pages of the sequences are
    done (after a prompt, or after ``inkling_kv_evict``).

    ``bounds [num_pages, kv_heads, 2, 128]`` bf16 (minima at ``[.., 0, :]``) is written in place, at
    those pages only; without it a new tensor is made, zero at all other pages.  Only slots that the
    sequence has filled count; a NaN among them makes the bound NaN.  A page that several sequences
    hold must be full in each of them (its bounds are otherwise those of one of them).
    ``max_seqlen_q`` (a host integer) sizes the grid and nothing else.  Returns ``bounds``."""
    if bounds is not None and _ops.USE_TORCH_OPS:
        outs = _lib.plain_call("page_bounds", k_cache, bounds, block_table, cu_seqlens_q,
                               cu_seqlens_k, max_seqlen_q or 0)
        if outs is not None:
            return bounds
    return _checked_bounds(k_cache, block_table, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, bounds)


@torch.no_grad()
def _checked_bounds(k_cache, block_table, cu_q, cu_k, max_seqlen_q, bounds):
    name = "kv_page_bounds"
    _ops.refuse_tracing(name)
    _paged.cache(name, "k_cache", k_cache)
    device, (pages, size, kv_heads, dim) = k_cache.device, k_cache.shape
    cu_q, cu_k, block_table = _paged.sequences(name, device, cu_q, cu_k, block_table)
    given = bounds
    if bounds is None:
        bounds = torch.zeros((pages, kv_heads, 2, dim), dtype=torch.bfloat16, device=device)
    _paged.page_bounds(name, bounds, kv_heads, pages, device)
    if not pages:
        return bounds
    p = _lib.PageBoundsParams()
    _paged.fill_seqs(p, cu_q, cu_k, block_table, size, pages)
    p.k_cache, p.bounds = k_cache.data_ptr(), bounds.data_ptr()
    _paged.fill_strides(p, k=(k_cache, ("page", "t", "h")), bounds=(bounds, ("page", "h")))
    p.kv_heads, p.head_dim, p.dtype = kv_heads, dim, _lib.IFA4_DTYPE_BF16
    p.max_seqlen_q = _paged.hint(max_seqlen_q)
    _paged.launch("page_bounds", p, device)
    _ops.written(given)
    return bounds


def inkling_kv_page_scores(q, bounds, rel_logits, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, rel_extent,
                           page_size, window_size=(-1, -1), *, block_table, softmax_scale=None,
                           first_pages=0, last_pages=0, out=None):
    """``scores [total_q, kv_heads, max_pages]`` fp32 (``max_pages`` as wide as ``block_table``): for
    every query, KV head and page an upper bound of the page's logits,

        max over the heads h of the group of
          softmax_scale * sum_i (max(q_i, 0) max_i + min(q_i, 0) min_i) + max over j of bias(h, p - j)

    over the page's visible keys ``j`` (``0 <= p - j``, and ``<= window_size[0]`` where that is not
    negative), with ``bias(h, d) = rel_logits[t, h, d]`` for ``d < rel_extent`` and 0 beyond.  A page
    without a visible key scores -inf; the first ``first_pages`` and the last ``last_pages`` of a
    query's visible pages score +inf, so they are always chosen.  NaN or infinite bounds give what the
    formula gives (a choice ranks NaN above everything).  A table entry that is no page counts as a
    page of zero keys, as the attention reads it.  Rows of no sequence (behind the last, or in front
    of the first where the offsets do not begin at 0) are -inf in a new tensor and stay as they are
    in ``out``."""
    if out is None and _ops.USE_TORCH_OPS:
        outs = _lib.plain_call("page_scores", q, bounds, rel_logits, cu_seqlens_q, cu_seqlens_k,
                               block_table, max_seqlen_q or 0, rel_extent, page_size,
                               -1 if window_size is None else window_size[0],
                               1.0 / _ops.HEAD_DIM if softmax_scale is None else softmax_scale,
                               first_pages, last_pages)
        if outs is not None:
            return outs[0]
    return _checked_scores(q, bounds, rel_logits, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
                           rel_extent, page_size, window_size, block_table, softmax_scale,
                           first_pages, last_pages, out)


@torch.no_grad()
def _checked_scores(q, bounds, rel_logits, cu_q, cu_k, max_seqlen_q, rel_extent, page_size,
                    window_size, block_table, softmax_scale, first_pages, last_pages, out):
    name = "kv_page_scores"
    _ops.refuse_tracing(name)
    _paged.page_bounds(name, bounds, None, None, None)
    device, pages, kv_heads = bounds.device, bounds.shape[0], bounds.shape[1]
    if kv_heads < 1:
        raise ValueError(f"{name}: bounds have no KV head")
    _paged.page_size(name, page_size)
    q, rel, rel_extent, scale = _paged.queries(name, q, rel_logits, kv_heads, rel_extent,
                                               softmax_scale, device)
    cu_q, cu_k, block_table = _paged.sequences(name, device, cu_q, cu_k, block_table)
    first_pages, last_pages = int(first_pages), int(last_pages)
    if not (0 <= first_pages < 1 << 31 and 0 <= last_pages < 1 << 31):
        raise ValueError(f"{name}: first_pages and last_pages must not be negative")
    shape = (q.shape[0], kv_heads, block_table.shape[1])
    given = out
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=device)
    else:
        _paged.tensor(name, "out", out, device, torch.float32, 3)
        if tuple(out.shape) != shape or (out.numel() and not _paged.rows_apart(out)):
            raise ValueError(f"{name}: out must be {list(shape)} with unit last stride and rows that "
                             "do not overlap")
    if out.numel():
        p = _lib.PageScoresParams()
        _paged.fill_seqs(p, cu_q, cu_k, block_table, page_size, pages)
        p.q, p.bounds, p.rel = q.data_ptr(), bounds.data_ptr(), rel.data_ptr()
        p.scores = out.data_ptr()
        _paged.fill_strides(p, q=(q, ("t", "h")), rel=(rel, ("t", "h")), scores=(out, ("t", "h")))
        # without a page nothing is read through these strides
        p.bounds_stride_page, p.bounds_stride_h = bounds.stride()[:2] if pages else (256, 256)
        p.total_q, p.n_heads, p.kv_heads = q.shape[0], q.shape[1], kv_heads
        p.head_dim, p.dtype = _ops.HEAD_DIM, _lib.IFA4_DTYPE_BF16
        p.rel_extent, p.softmax_scale = rel_extent, scale
        p.window_left, p.max_seqlen_q = _paged.window(window_size), _paged.hint(max_seqlen_q)
        p.first_pages, p.last_pages = first_pages, last_pages
        p.zero_padding = int(given is None)
        _paged.launch("page_scores", p, device)
    _ops.written(given)
    return out


def inkling_kv_select_pages(scores, num_selected, *, out=None):
    """``[total_q, kv_heads, num_selected]`` int32: the places of the ``num_selected`` largest of every
    row of ``scores [total_q, kv_heads, max_pages]`` fp32, ascending.  Of equal scores at the border
    the lowest places are taken, NaN ranks above everything, -inf is never taken; a row with fewer
    choices ends in -1.  ``out`` is other memory than ``scores``."""
    if out is None and _ops.USE_TORCH_OPS:
        outs = _lib.plain_call("select_pages", scores, num_selected)
        if outs is not None:
            return outs[0]
    return _checked_select(scores, num_selected, out)


@torch.no_grad()
def _checked_select(scores, num_selected, out):
    name = "kv_select_pages"
    _ops.refuse_tracing(name)
    _paged.tensor(name, "scores", scores, None, torch.float32, 3)
    num_selected = int(num_selected)
    if not 1 <= num_selected <= _paged.MOST:
        raise ValueError(f"{name}: num_selected must be in [1, 2^26]")
    rows, heads, width = scores.shape
    if scores.numel() and scores.stride(2) != 1:
        scores = scores.contiguous()
    shape, given = (rows, heads, num_selected), out
    if out is None:
        out = torch.empty(shape, dtype=torch.int32, device=scores.device)
    else:
        _paged.tensor(name, "out", out, scores.device, torch.int32, 3)
        if tuple(out.shape) != shape or (out.numel() and not _paged.rows_apart(out)):
            raise ValueError(f"{name}: out must be {list(shape)} with unit last stride and rows that "
                             "do not overlap")
    if out.numel():
        p = _lib.SelectPagesParams()
        p.scores, p.pages = scores.data_ptr(), out.data_ptr()
        _paged.fill_strides(p, scores=(scores, ("t", "h")), pages=(out, ("t", "h")))
        p.rows, p.kv_heads, p.width, p.num_selected = rows, heads, width, num_selected
        _paged.launch("select_pages", p, scores.device)
    _ops.written(given)
    return out


def inkling_fa4_rel_attention_decode_pages(q, k, v, rel_logits, cu_seqlens_q, cu_seqlens_k,
                                           max_seqlen_q, max_seqlen_k, rel_extent, pages,
                                           window_size=(-1, -1), n_heads=None, kv_heads=None,
                                           head_dim=128, *, block_table, softmax_scale=None, out=None,
                                           num_splits=0, workspace=None, return_lse=False, lse=None):
    """Attention of every query to the keys of its chosen pages: the result of
    ``inkling_fa4_rel_attention_triton(..., causal_align="bottom_right", block_table=block_table)``
    with the keys of all other pages masked.

    ``pages [total_q, kv_heads, num_selected]`` int32 are indices into the query's row of
    ``block_table`` (page ``c`` holds positions ``c * page_size ..``), one list for each query and KV
    head, in any order.  An entry below 0, past the query's last page or without a visible key adds
    nothing; one that is listed twice counts twice.  Positions, causal mask, window and relative bias
    are those of the whole sequence.  Where every visible page is listed once, this is the attention
    itself.

    Any number of queries a sequence (each reads its own pages: for long chunks that share their keys
    the prefill does less).  A query without keys gets 0 (lse -inf); one whose logits hold NaN or +inf
    is NaN.  Rows of no sequence are zeros (lse -inf) in new tensors and stay as they are in ``out`` /
    ``lse`` where ``out`` is given.  ``num_splits``: CTAs that share a query's pages (0:
    automatic); ``workspace``: a reusable uint8 CUDA tensor (allocated per call when absent or too
    small); calls that may run at the same time need one each.  Logits, weights and sums are held in 32
    bits, the weights to 16 in the product with ``v``; the output's is the only other rounding."""
    if (out is None and lse is None and not return_lse and n_heads is None and kv_heads is None
            and head_dim == _ops.HEAD_DIM and _ops.USE_TORCH_OPS):
        outs = _lib.plain_call("decode_pages", q, k, v, rel_logits, cu_seqlens_q, cu_seqlens_k, pages,
                               block_table, workspace, rel_extent,
                               -1 if window_size is None else window_size[0], max_seqlen_k or 0,
                               1.0 / _ops.HEAD_DIM if softmax_scale is None else softmax_scale,
                               num_splits)
        if outs is not None:
            return outs[0]
    return _checked_decode(q, k, v, rel_logits, cu_seqlens_q, cu_seqlens_k, max_seqlen_k, rel_extent,
                           pages, window_size, n_heads, kv_heads, head_dim, block_table,
                           softmax_scale, out, num_splits, workspace, return_lse, lse)


@torch.no_grad()
def _checked_decode(q, k, v, rel_logits, cu_q, cu_k, max_seqlen_k, rel_extent, pages, window_size,
                    n_heads, kv_heads, head_dim, block_table, softmax_scale, out, num_splits,
                    workspace, return_lse, lse):
    name = "decode_pages"
    _ops.refuse_tracing(name)
    if block_table is None:
        raise ValueError(f"{name}: needs a paged cache (block_table)")
    _paged.cache(name, "k", k)
    _paged.cache(name, "v", v, k.device)
    cu_q, cu_k, block_table = _paged.sequences(name, k.device, cu_q, cu_k, block_table)
    given = (out, lse)
    _paged.distances(name, int(rel_extent))
    q, k, v, rel, out, n_heads, kv_heads, rel_extent, window_left, scale = _ops._prepare(
        name, q, k, v, rel_logits, cu_q, cu_k, rel_extent, True, window_size, n_heads, kv_heads,
        head_dim, softmax_scale, "bottom_right", out, block_table)
    if any(s <= 0 for s in out.stride()[:-1]) and out.numel():
        raise ValueError(f"{name}: out must not be an expanded tensor")
    lse = _ops._lse_buffer(q, n_heads, return_lse, lse)
    if scale == math.inf:
        raise ValueError(f"{name}: softmax_scale must be finite")
    _paged.tensor(name, "pages", pages, q.device, torch.int32, 3)
    if pages.shape[:2] != (q.shape[0], kv_heads) or pages.shape[2] > _paged.MOST:
        raise ValueError(f"{name}: pages must be [total_q, kv_heads, num_selected], got "
                         f"{tuple(pages.shape)}")
    if pages.numel() and pages.stride(2) != 1:
        pages = pages.contiguous()
    if workspace is not None and not (isinstance(workspace, torch.Tensor)
                                      and workspace.device == q.device
                                      and workspace.is_contiguous()):
        raise ValueError(f"{name}: workspace must be a contiguous tensor on q's device")
    if workspace is not None and workspace.data_ptr() % 16:
        raise ValueError(f"{name}: workspace must be 16-byte aligned")
    if q.numel() == 0:
        return (out, lse) if lse is not None else out
    if k.shape[0] == 0:
        raise ValueError(f"{name}: the cache has no pages")
    p = _lib.DecodePagesParams()
    p.decode = _ops._decode_params(q, k, v, rel, out, cu_q, cu_k, n_heads, kv_heads, rel_extent, True,
                                   min(window_left, 0x7fffffff), "bottom_right",
                                   _paged.hint(max_seqlen_k), scale, num_splits, 0, block_table)
    _ops._fill_lse(p.decode, lse)
    p.pages = pages.data_ptr()
    p.pages_stride_t, p.pages_stride_h = pages.stride()[:2]
    p.num_selected, p.table_width = pages.shape[2], block_table.shape[1]
    p.zero_padding = int(given[0] is None)
    _paged.launch(name, p, q.device, workspace, sized=True)
    _ops.written(*given)
    return (out, lse) if lse is not None else out


__all__ = ["inkling_kv_page_bounds", "inkling_kv_page_scores", "inkling_kv_select_pages",
           "inkling_fa4_rel_attention_decode_pages"]
