"""Eviction from a paged cache by the attention weight that keys have gathered: the weights of a call's
queries, summed for every key, and the compaction of each sequence to a budget of keys.  The calls are
no dispatcher operators and not differentiable; under ``make_fx`` and ``torch.jit.trace`` they are
refused."""
from __future__ import annotations

import torch

from . import _lib, _ops, _paged


def inkling_kv_attention_mass(q, k, rel_logits, lse, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
                              max_seqlen_k, rel_extent, window_size=(-1, -1), *, block_table,
                              softmax_scale=None, mass=None):
    """``mass[b, g, j]``: the sum of the attention weights that key ``j`` of sequence ``b`` gets from
    the sequence's queries, over the heads of group ``g``,

        sum over t, h of exp(softmax_scale * q[t, h] . k[j, g] + bias(t, h, p - j) - lse[h, t])

    over the queries that see it (``causal_align="bottom_right"``, the window, the relative bias as in
    the attention), in fp32 and in a fixed order.  ``lse [n_heads, total_q]`` fp32 is what the
    attention call on the same arguments (with ``causal_align="bottom_right"``) returns with
    ``return_lse=True``; a query whose lse is -inf (one without keys, or padding for which the caller
    sets it) adds nothing, whatever it holds.

    ``k`` is the paged cache.  ``mass [batch, kv_heads, width]`` fp32 with unit last stride is added to
    in place, at the places of the sequences' keys only (a key from ``width`` on has none); without it
    a new tensor ``max_pages * page_size`` wide is made, zero behind a sequence's keys.  Any number of
    queries: the whole prompt, its last ones, or a new token each step.  At most 128 query heads per KV
    head.  ``max_seqlen_q`` and ``max_seqlen_k`` (host integers) size the grid and nothing else.
    Returns the masses."""
    if _ops.USE_TORCH_OPS:
        outs = _lib.plain_call("attention_mass", q, k, rel_logits, lse, cu_seqlens_q, cu_seqlens_k,
                               block_table, mass, rel_extent,
                               -1 if window_size is None else window_size[0], max_seqlen_q or 0,
                               max_seqlen_k or 0,
                               1.0 / _ops.HEAD_DIM if softmax_scale is None else softmax_scale)
        if outs is not None:
            return outs[0] if mass is None else mass
    return _checked_mass(q, k, rel_logits, lse, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
                         max_seqlen_k, rel_extent, window_size, block_table, softmax_scale, mass)


def _places(name, t, batch, kv_heads, device, what):
    _paged.tensor(name, what, t, device, torch.float32, 3)
    if t.shape[:2] != (batch, kv_heads) or t.shape[2] > 1 << 30:
        raise ValueError(f"{name}: {what} must be [batch, kv_heads, width], got {tuple(t.shape)}")


@torch.no_grad()
def _checked_mass(q, k, rel_logits, lse, cu_q, cu_k, max_seqlen_q, max_seqlen_k, rel_extent,
                  window_size, block_table, softmax_scale, mass):
    name = "kv_attention_mass"
    _ops.refuse_tracing(name)
    _paged.cache(name, "k", k)
    device, (pages, size, kv_heads, dim) = k.device, k.shape
    q, rel, rel_extent, scale = _paged.queries(name, q, rel_logits, kv_heads, rel_extent,
                                               softmax_scale, device)
    if q.shape[1] // kv_heads > 128:
        raise ValueError(f"{name}: at most 128 query heads per KV head")
    cu_q, cu_k, block_table = _paged.sequences(name, device, cu_q, cu_k, block_table)
    batch = cu_q.numel() - 1
    _paged.tensor(name, "lse", lse, device, torch.float32, 2)
    if lse.shape != (q.shape[1], q.shape[0]):
        raise ValueError(f"{name}: lse must be [n_heads, total_q], got {tuple(lse.shape)}")
    given = mass
    if mass is None:
        width = block_table.shape[1] * size
        if width > 1 << 30:
            raise ValueError(f"{name}: a mass of {width} places (the table's) is too wide; give one")
        mass = torch.empty((batch, kv_heads, width), dtype=torch.float32, device=device)
    else:
        _places(name, mass, batch, kv_heads, device, "mass")
        if mass.numel() and not _paged.rows_apart(mass):
            raise ValueError(f"{name}: mass must have unit last stride and rows that do not overlap")
    if not mass.numel():
        return mass
    if pages == 0:
        raise ValueError(f"{name}: the cache has no pages")
    p = _lib.AttentionMassParams()
    _paged.fill_seqs(p, cu_q, cu_k, block_table, size, pages)
    p.q, p.k_cache, p.rel = q.data_ptr(), k.data_ptr(), rel.data_ptr()
    p.lse, p.mass = lse.data_ptr(), mass.data_ptr()
    _paged.fill_strides(p, q=(q, ("t", "h")), k=(k, ("page", "t", "h")), rel=(rel, ("t", "h")),
                        lse=(lse, ("h", "t")), mass=(mass, ("b", "h")))
    p.total_q, p.n_heads, p.kv_heads = q.shape[0], q.shape[1], kv_heads
    p.head_dim, p.dtype = dim, _lib.IFA4_DTYPE_BF16
    p.rel_extent, p.softmax_scale = rel_extent, scale
    p.window_left = _paged.window(window_size)
    p.max_seqlen_q, p.max_seqlen_k = _paged.hint(max_seqlen_q), _paged.hint(max_seqlen_k)
    p.mass_width, p.accumulate = mass.shape[2], int(given is not None)
    _paged.launch("attention_mass", p, device)
    _ops.written(given)
    return mass


def inkling_kv_evict(k_cache, v_cache, mass, block_table, cu_seqlens_k, budget, *, first=0, recent=0):
    """Cuts every sequence of more than ``budget`` keys down to ``budget``, for each KV head on its
    own: the first ``first`` keys and the last ``recent`` stay, and of the others those of the largest
    ``mass [batch, kv_heads, width]`` (of equal ones at the border the first; NaN ranks above
    everything; a key from ``width`` on has the mass 0).  What stays moves, in its order, to the places
    ``0 .. budget - 1`` of the sequence, in place in ``k_cache`` and ``v_cache``; shorter sequences
    stay as they are.

    Returns ``(kept, mass, cu_seqlens_k)``: ``kept [batch, kv_heads, budget]`` int32, the places that
    the keys had (-1 behind the last); the masses of what stays, zero behind it, in a new tensor like
    ``mass``; and the offsets of the new lengths, with which the following calls are made (pages past
    them are free).

    With ``recent >= rel_extent - 1`` the relative bias of a query that comes next is what it would
    have been: the keys within its reach keep their distances, and older ones have no bias at either
    place.  (A layer with a window keeps its recent keys by it instead: distances beyond ``recent``
    change.)  The keys keep the rotation they were appended with; new tokens of a model with rotation
    take it from ``inkling_qk_norm_rope`` with the offsets before the eviction and are appended
    without one.  Bounds of pages (``inkling_kv_page_bounds``) have to be made anew.

    ``k_cache`` and ``v_cache`` are two tensors, or slices of one without an element in common (with the
    same strides, or in turn; others are refused).  No page that keys move into or out of may be held by
    another sequence, or twice by its own (the first ``first`` keys stay where they are, so pages full
    of them may be shared).  A kept key whose table entry is no page becomes zeros at its new place, and
    nothing is written to a place without a page."""
    if _ops.USE_TORCH_OPS:
        outs = _lib.plain_call("kv_evict", k_cache, v_cache, mass, block_table, cu_seqlens_k, budget,
                               first, recent)
        if outs is not None:
            return outs
    return _checked_evict(k_cache, v_cache, mass, block_table, cu_seqlens_k, budget, first, recent)


@torch.no_grad()
def _checked_evict(k_cache, v_cache, mass, block_table, cu_k, budget, first, recent):
    name = "kv_evict"
    _ops.refuse_tracing(name)
    _paged.cache(name, "k_cache", k_cache)
    device, (pages, size, kv_heads, dim) = k_cache.device, k_cache.shape
    _paged.cache(name, "v_cache", v_cache, device)
    if v_cache.shape != k_cache.shape:
        raise ValueError(f"{name}: k_cache and v_cache differ in shape")
    if v_cache.data_ptr() == k_cache.data_ptr() and k_cache.numel():
        raise ValueError(f"{name}: k_cache and v_cache are the same memory")
    _, cu_k, block_table = _paged.sequences(name, device, cu_k, cu_k, block_table)
    batch = cu_k.numel() - 1
    _places(name, mass, batch, kv_heads, device, "mass")
    budget, first, recent = int(budget), int(first), int(recent)
    if not 1 <= budget <= 1 << 30 or first < 0 or recent < 0 or first + recent > budget:
        raise ValueError(f"{name}: budget must be in [1, 2^30] and hold the first and the recent keys")
    if mass.numel() and (mass.stride(2) != 1 and mass.shape[2] > 1 or min(mass.stride()) < 0):
        mass = mass.contiguous()
    kept = torch.empty((batch, kv_heads, budget), dtype=torch.int32, device=device)
    left = torch.empty(mass.shape, dtype=torch.float32, device=device)
    cu_out = torch.empty(batch + 1, dtype=torch.int32, device=device)
    p = _lib.KvEvictParams()
    _paged.fill_seqs(p, cu_k, cu_k, block_table, size, pages)
    p.k_cache, p.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    p.mass, p.mass_out = mass.data_ptr(), left.data_ptr()
    p.kept, p.cu_out = kept.data_ptr(), cu_out.data_ptr()
    if pages:
        _paged.fill_strides(p, k=(k_cache, ("page", "t", "h")), v=(v_cache, ("page", "t", "h")))
    else:  # nothing is moved through these strides
        for nm in ("k_stride_page", "k_stride_t", "k_stride_h", "v_stride_page", "v_stride_t",
                   "v_stride_h"):
            setattr(p, nm, dim)
    _paged.fill_strides(p, mass=(mass, ("b", "h")), mass_out=(left, ("b", "h")))
    p.kv_heads, p.head_dim, p.mass_width = kv_heads, dim, mass.shape[2]
    p.budget, p.first, p.recent = budget, first, recent
    p.dtype = _lib.IFA4_DTYPE_BF16
    _paged.launch(name, p, device, sized=True)
    _ops.written(k_cache, v_cache)
    return kept, left, cu_out


__all__ = ["inkling_kv_attention_mass", "inkling_kv_evict"]
