"""CPU oracle in 64 bits for the long-context operators over the paged cache (TEST INFRASTRUCTURE
ONLY): bounds of pages, scores of pages, the choice of the largest, attention over chosen pages,
gathered attention weight and eviction.  Parity unpinned: the reference has none of them, so these
functions state the formulas in include/inkling_fa4.h, one row at a time, each beside the size of the
terms that its fp32 error grows with."""
from __future__ import annotations

import numpy as np

__all__ = ["page_bounds", "page_scores", "select_largest", "row_place", "decode_pages",
           "attention_mass", "kv_evict"]


def _place(table_row, j, page_size, num_pages):
    """(page, slot) of key j, or None."""
    c = j // page_size
    if c >= len(table_row) or not 0 <= table_row[c] < num_pages:
        return None
    return int(table_row[c]), j % page_size


def _rows(cache, table_row, places, head):
    """Cache rows [len(places), 128] in float64; zeros where there is no page."""
    out = np.zeros((len(places), cache.shape[-1]))
    for i, j in enumerate(places):
        at = _place(table_row, int(j), cache.shape[1], cache.shape[0])
        if at is not None:
            out[i] = cache[at[0], at[1], head]
    return out


def row_place(cu_q, cu_k, t):
    """(sequence, position) of row t, or None for a row of no sequence."""
    for b in range(len(cu_q) - 1):
        if cu_q[b] <= t < cu_q[b + 1]:
            return b, int(cu_k[b + 1] - cu_k[b]) - int(cu_q[b + 1] - cu_q[b]) + int(t - cu_q[b])
    return None


def page_bounds(bounds, k_cache, table, cu_q, cu_k):
    out = bounds.copy()
    ps = k_cache.shape[1]
    for b in range(len(cu_q) - 1):
        n_q, n_k = int(cu_q[b + 1] - cu_q[b]), int(cu_k[b + 1] - cu_k[b])
        if n_q <= 0 or n_k <= 0:
            continue
        for c in range(max(0, n_k - n_q) // ps, (n_k - 1) // ps + 1):
            at = _place(table[b], c * ps, ps, k_cache.shape[0])
            if at is not None:
                keys = k_cache[at[0], :min(ps, n_k - c * ps)]
                out[at[0], :, 0], out[at[0], :, 1] = keys.min(0), keys.max(0)
    return out


def _bias(rel_row, d, extent):
    """Bias [heads, len(d)] at distances d >= 0."""
    near = d < extent
    return np.where(near, rel_row[:, np.where(near, d, 0)], 0.0)


def _size(x):
    """Sizes of terms that are added up; what swallows or hides the others has no rounding of its own."""
    x = np.abs(x)
    return np.where(x < 1e30, x, 0.0)


def page_scores(q, bounds, rel, cu_q, cu_k, table, page_size, extent, window, scale, first=0, last=0):
    """Scores and, for each, the sum of the sizes of its products (times scale)."""
    T, H, _ = q.shape
    K, P = bounds.shape[1], table.shape[1]
    G = H // K
    out, size = np.full((T, K, P), -np.inf), np.zeros((T, K, P))
    for t in range(T):
        at = row_place(cu_q, cu_k, t)
        if at is None or at[1] < 0:
            continue
        b, p = at
        lo = max(0, p - window) if window >= 0 else 0
        for c in range(lo // page_size, min(P, p // page_size + 1)):
            page = table[b, c]
            ends = bounds[page] if 0 <= page < len(bounds) else np.zeros(bounds.shape[1:])
            j = np.arange(max(lo, c * page_size), min(p, (c + 1) * page_size - 1) + 1)
            bias = _bias(rel[t], p - j, extent).max(1)
            for g in range(K):
                x = q[t, g * G:(g + 1) * G]
                dot = np.maximum(x, 0) @ ends[g, 1] + np.minimum(x, 0) @ ends[g, 0]
                terms = _size(x) @ _size(ends[g]).max(0)
                s = dot * scale + bias[g * G:(g + 1) * G]
                out[t, g, c] = np.nan if np.isnan(s).any() else s.max()
                size[t, g, c] = (terms * scale + _size(bias[g * G:(g + 1) * G])).max()
            if c - lo // page_size < first or p // page_size - c < last:
                out[t, :, c] = np.inf
    return out, size


def select_largest(x, count, always=()):
    """Places of the `count` largest of a vector, ascending; -inf never, NaN above everything,
    `always` above that, the lowest places of equal ones."""
    def rank(i):
        if i in always:
            return (2, 0.0)
        return (1, 0.0) if np.isnan(x[i]) else (0, float(x[i]))
    able = [i for i in range(len(x)) if i in always or not x[i] == -np.inf]
    able.sort(key=lambda i: (-rank(i)[0], -rank(i)[1], i))
    return sorted(able[:count])


def decode_pages(q, k_cache, v_cache, rel, cu_q, cu_k, table, pages, extent, window, scale):
    """Outputs, their sums of |p v| / sum of p, log-sum-exps, and the sizes of the logits' terms."""
    T, H, D = q.shape
    ps, K = k_cache.shape[1], k_cache.shape[2]
    G = H // K
    out, weight = np.zeros((T, H, D)), np.zeros((T, H, D))
    lse, size = np.full((H, T), -np.inf), np.zeros((T, H))
    for t in range(T):
        at = row_place(cu_q, cu_k, t)
        if at is None:
            continue
        b, p = at
        lo = max(0, p - window) if window >= 0 else 0
        for g in range(K):
            j = [c * ps + i for c in pages[t, g].tolist() if c >= 0 for i in range(ps)
                 if lo <= c * ps + i <= p]
            if not j:
                continue
            j = np.array(j)
            k, v = _rows(k_cache, table[b], j, g), _rows(v_cache, table[b], j, g)
            heads = slice(g * G, (g + 1) * G)
            with np.errstate(invalid="ignore", over="ignore"):
                bias = _bias(rel[t, heads], p - j, extent)
                x = q[t, heads] @ k.T * scale + bias
                m = x.max(1, keepdims=True)
                e = np.exp(x - np.where(m == -np.inf, 0.0, m))
                s = e.sum(1, keepdims=True)
                out[t, heads] = np.where(s == 0, 0.0, e @ v / np.where(s == 0, 1.0, s))
                weight[t, heads] = e @ np.abs(v) / np.where(s == 0, 1.0, s)
                lse[heads, t] = np.where(s == 0, -np.inf, m + np.log(s))[:, 0]
                size[t, heads] = (_size(q[t, heads]) @ _size(k).T * scale + _size(bias)).max(1)
    return out, weight, lse, size


def attention_mass(mass, q, k_cache, rel, lse, cu_q, cu_k, table, extent, window, scale):
    """Masses, and a bound on the fp32 error of each: the sum over its terms of the weight times the
    size of what is added up in its exponent."""
    out, err = mass.astype(np.float64).copy(), np.zeros(mass.shape)
    H, K = q.shape[1], k_cache.shape[2]
    G = H // K
    for b in range(len(cu_q) - 1):
        n_q, n_k = int(cu_q[b + 1] - cu_q[b]), int(cu_k[b + 1] - cu_k[b])
        n = min(n_k, mass.shape[2])
        if n_q <= 0 or n <= 0:
            continue
        for g in range(K):
            k = _rows(k_cache, table[b], np.arange(n), g)
            for t in range(int(cu_q[b]), int(cu_q[b + 1])):
                p = n_k - n_q + t - int(cu_q[b])
                d = p - np.arange(n)
                seen = (d >= 0) & ((d <= window) if window >= 0 else True)
                for h in range(g * G, (g + 1) * G):
                    if lse[h, t] == -np.inf:
                        continue
                    with np.errstate(invalid="ignore", over="ignore"):
                        bias = _bias(rel[t, h:h + 1], np.maximum(d, 0), extent)[0]
                        x = k @ q[t, h] * scale + bias - lse[h, t]
                        e = np.where(seen, np.exp(x), 0.0)
                        out[b, g, :n] += e
                        size = _size(k) @ _size(q[t, h]) * scale + _size(bias) + _size(lse[h, t])
                        err[b, g, :n] += e * np.where(seen, size, 0.0)
    return out, err


def kv_evict(k_cache, v_cache, mass, table, cu_k, budget, first, recent):
    """(k_cache, v_cache, kept, mass, cu_k) after the eviction."""
    B, K, W = mass.shape
    ps, pages = k_cache.shape[1], k_cache.shape[0]
    caches = [k_cache.copy(), v_cache.copy()]
    kept, left = np.full((B, K, budget), -1, np.int32), np.zeros_like(mass)
    cu = np.zeros(B + 1, np.int32)
    for b in range(B):
        n = max(0, int(cu_k[b + 1] - cu_k[b]))
        cu[b + 1] = cu[b] + min(n, budget)
        for g in range(K):
            x = np.zeros(n, mass.dtype)
            x[:min(n, W)] = mass[b, g, :n]
            stay = list(range(n))
            if n > budget:
                low = np.where(x == -np.inf, np.float64(-1e300), x.astype(np.float64))
                stay = select_largest(low, budget, {i for i in range(n) if i < first or i >= n - recent})
            for to, at in enumerate(stay):
                kept[b, g, to] = at
                if to < W:
                    left[b, g, to] = x[at]
                if n > budget and to != at:
                    dst, src = _place(table[b], to, ps, pages), _place(table[b], at, ps, pages)
                    if dst is None:
                        continue
                    for new, old in zip(caches, (k_cache, v_cache)):
                        new[dst[0], dst[1], g] = 0.0 if src is None else old[src[0], src[1], g]
    return caches[0], caches[1], kept, left, cu
