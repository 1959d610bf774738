"""CPU oracle in 64 bits for the operators next to the attention (TEST INFRASTRUCTURE ONLY): norm
and rotation of query and key heads with their gradients, the append to a paged cache, decode
attention through a page table, and the bias by distance buckets.  Parity unpinned: the reference
repository has these steps only as boxes of its diagram (outputs/architecture.md:18-64, :117-120) or
not at all, so these functions state the formulas in include/inkling_fa4.h."""
from __future__ import annotations

import numpy as np

from .rel_logits_oracle import token_positions

__all__ = ["norm_rope", "norm_rope_pair_size", "norm_rope_grads", "kv_append", "decode_paged",
           "bucket_of", "bucket_bias", "bucket_bias_grad"]


def _pairs(rotary_dim, interleaved):
    i = np.arange(rotary_dim // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)


def _rotate(y, pos, inv_freq, interleaved, sign=1.0):
    if inv_freq is None:
        return y
    inv_freq = np.asarray(inv_freq, np.float64)
    angle = np.asarray(pos, np.float64)[:, None, None] * inv_freq
    c, s = np.cos(angle), sign * np.sin(angle)
    a, b = _pairs(2 * len(inv_freq), interleaved)
    out = y.copy()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def norm_rope(x, weight, pos, eps, inv_freq, interleaved):
    """``x [tokens, heads, 128]`` -> normalised (eps None: not) and rotated rows, float64."""
    y = np.asarray(x, np.float64)
    if eps is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
        if weight is not None:
            y = y * np.asarray(weight, np.float64)
    return _rotate(y, pos, inv_freq, interleaved)


def norm_rope_pair_size(y, inv_freq, interleaved):
    """Per element, the length of the pair it belongs to (its own size outside the rotation): the
    scale of the fp32 error of a rotated value."""
    size = np.abs(y)
    if inv_freq is not None:
        a, b = _pairs(2 * len(inv_freq), interleaved)
        both = np.hypot(y[..., a], y[..., b])
        size[..., a] = both
        size[..., b] = both
    return size


def norm_rope_grads(dout, x, weight, pos, eps, inv_freq, interleaved):
    """Gradients ``(dx, dw)`` and the sizes of the sums behind them ``(dx_size, dw_size)``."""
    x = np.asarray(x, np.float64)
    g = _rotate(np.asarray(dout, np.float64), pos, inv_freq, interleaved, -1.0)
    gs = norm_rope_pair_size(g, inv_freq, interleaved)
    if eps is None:
        return g, None, gs, None
    w = np.ones(x.shape[-1]) if weight is None else np.asarray(weight, np.float64)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xhat = x * r
    dw, dw_size = (g * xhat).sum((0, 1)), (gs * np.abs(xhat)).sum((0, 1))
    gw = g * w
    dx = r * (gw - xhat * (gw * xhat).mean(-1, keepdims=True))
    size = r * (gs * np.abs(w) + np.abs(xhat) * (gs * np.abs(w * xhat)).mean(-1, keepdims=True))
    return dx, dw, size, dw_size


def kv_append(k_cache, v_cache, k_rows, v_rows, table, cu_q, cu_k):
    """Writes rows into copies of the caches; rows without a place write nothing."""
    k_cache, v_cache = k_cache.copy(), v_cache.copy()
    num_pages, page_size = k_cache.shape[:2]
    cu_q = np.asarray(cu_q)
    pos = token_positions(k_rows.shape[0], cu_q, cu_k)
    for b in range(len(cu_q) - 1):
        for t in range(cu_q[b], min(cu_q[b + 1], k_rows.shape[0])):
            p = pos[t]
            if p < 0 or p // page_size >= table.shape[1]:
                continue
            page = table[b, p // page_size]
            if 0 <= page < num_pages:
                k_cache[page, p % page_size] = k_rows[t]
                v_cache[page, p % page_size] = v_rows[t]
    return k_cache, v_cache


def decode_paged(q, k_cache, v_cache, rel, lens, table, scale, rel_extent, window_left=-1):
    """Decode with the query at the last position of its ``lens[b]`` keys.  Returns the output
    [batch, heads, 128], the natural-log sum of exponentials [heads, batch], and the sum of
    weights times |v| (the scale of the output's error).  No visible key: 0 and -inf."""
    q, rel = np.asarray(q, np.float64), np.asarray(rel, np.float64)
    B, H, D = q.shape
    page_size, K = k_cache.shape[1:3]
    out, size = np.zeros((B, H, D)), np.zeros((B, H, D))
    lse = np.full((H, B), -np.inf)
    for b in range(B):
        n = int(lens[b])
        j = np.arange(n)
        d = n - 1 - j
        j, d = (j, d) if window_left < 0 else (j[d <= window_left], d[d <= window_left])
        if len(j) == 0:
            continue
        page, slot = table[b, j // page_size], j % page_size
        for h in range(H):
            k = k_cache[page, slot, h // (H // K)].astype(np.float64)
            v = v_cache[page, slot, h // (H // K)].astype(np.float64)
            x = k @ q[b, h] * scale
            near = d < rel_extent
            x[near] += rel[b, h, d[near]]
            m = x.max()
            p = np.exp(x - m)
            lse[h, b] = m + np.log(p.sum())
            p /= p.sum()
            out[b, h], size[b, h] = p @ v, p @ np.abs(v)
    return out, lse, size


def bucket_of(starts, rel_extent):
    """Bucket of every distance: the last one whose start is <= d, the first if there is none."""
    return np.maximum(np.searchsorted(np.asarray(starts), np.arange(rel_extent), side="right") - 1,
                      0)


def bucket_bias(table, starts, rel_extent):
    """``[heads, rel_extent]`` float64."""
    return np.asarray(table, np.float64)[bucket_of(starts, rel_extent)].T


def bucket_bias_grad(drel, starts, tokens=None):
    """Gradient ``[buckets, heads]`` of the table and the sums of |drel| behind it."""
    drel = np.asarray(drel, np.float64)[:tokens]
    onehot = np.eye(len(starts))[bucket_of(starts, drel.shape[2])]
    return (drel.sum(0) @ onehot).T, (np.abs(drel).sum(0) @ onehot).T
