"""The operators of long contexts over the paged cache, in their plain form and as the package's
calls, over the sizes they meet: bounds of a page's keys, scores of pages for a query, the choice
of pages, attention over the chosen pages; the attention weight that each key has gathered, and
the eviction of the keys with the least.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed, ``run``
is one call (``own`` false: elementary torch operations in 32 bits or more; ``own`` true: the
package's entry points), ``exact`` the same outputs in 64 bits from the definitions, ``work``
the bytes and operations one call cannot do without."""
import math
import os
import random
import sys

import torch

own = False

HEAD_DIM = 128
_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "inkling-fa4-relative-attention_b200")


def _package():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import inkling_fa4
    return inkling_fa4


# --- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # one new token a sequence: the page it went to gets new bounds (latency)
        {"name": "bounds_decode_b64", "kind": "bounds", "batch": 64, "chunk": 1, "lo": 4096,
         "hi": 32768, "kv_heads": 8, "heads": 32, "page_size": 16, "shape_seed": 0},
        # after a prompt of long sequences: the bounds of all their pages
        {"name": "bounds_prompt_8x32k", "kind": "bounds", "batch": 8, "chunk": 0, "lo": 32000,
         "hi": 32768, "kv_heads": 8, "heads": 32, "page_size": 64, "shape_seed": 1},
        # one sequence generating one token behind a long context (latency)
        {"name": "scores_b1_32k", "kind": "scores", "batch": 1, "chunk": 1, "lo": 32768,
         "hi": 32768, "heads": 32, "kv_heads": 8, "page_size": 16, "rel_extent": 128,
         "window": -1, "shape_seed": 2},
        # a decode batch of long contexts, a layer with the longest bias
        {"name": "scores_b64_32k", "kind": "scores", "batch": 64, "chunk": 1, "lo": 8192,
         "hi": 32768, "heads": 32, "kv_heads": 8, "page_size": 16, "rel_extent": 1024,
         "window": -1, "shape_seed": 3},
        # the choice for one token (latency)
        {"name": "select_b1_2k", "kind": "select", "rows": 1, "kv_heads": 8, "pages": 2048,
         "selected": 64, "shape_seed": 4},
        # the choice for a decode batch behind 131072 keys
        {"name": "select_b128_8k", "kind": "select", "rows": 128, "kv_heads": 8, "pages": 8192,
         "selected": 256, "shape_seed": 5},
        # one token over 64 of 2048 pages (latency)
        {"name": "sparse_b1_64p", "kind": "sparse", "batch": 1, "chunk": 1, "lo": 32768,
         "hi": 32768, "heads": 32, "kv_heads": 8, "page_size": 16, "selected": 64,
         "rel_extent": 128, "window": -1, "shape_seed": 6},
        # a decode batch over 4096 keys of each sequence's
        {"name": "sparse_b64_256p", "kind": "sparse", "batch": 64, "chunk": 1, "lo": 8192,
         "hi": 32768, "heads": 32, "kv_heads": 8, "page_size": 16, "selected": 256,
         "rel_extent": 1024, "window": -1, "shape_seed": 7},
        # the weights that one new token of each sequence gave (odd lengths)
        {"name": "mass_decode_b8", "kind": "mass", "batch": 8, "chunk": 1, "lo": 4097,
         "hi": 32767, "heads": 32, "kv_heads": 8, "page_size": 16, "rel_extent": 128,
         "window": -1, "gathered": True, "shape_seed": 8},
        # the weights of a whole prompt
        {"name": "mass_prompt_32k", "kind": "mass", "batch": 1, "chunk": 32768, "lo": 32768,
         "hi": 32768, "heads": 32, "kv_heads": 8, "page_size": 64, "rel_extent": 1024,
         "window": -1, "gathered": False, "shape_seed": 9},
        # a short cache that has to give up three quarters (latency)
        {"name": "evict_b1_4k", "kind": "evict", "batch": 1, "lo": 4096, "hi": 4096, "heads": 32,
         "kv_heads": 8, "page_size": 16, "budget": 1024, "first": 4, "recent": 128,
         "shape_seed": 10},
        # a batch of long contexts cut to a quarter, the recent ones as far as the longest bias
        {"name": "evict_b16_32k", "kind": "evict", "batch": 16, "lo": 30000, "hi": 32768,
         "heads": 32, "kv_heads": 8, "page_size": 64, "budget": 8192, "first": 4, "recent": 1024,
         "shape_seed": 11},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["bounds", "scores", "select", "sparse", "mass", "evict"])
    heads, kv_heads = rng.choice([(4, 4), (8, 2), (12, 4), (32, 8), (16, 16), (5, 1)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads,
            "shape_seed": rng.randrange(1 << 20)}
    if kind == "select":
        pages = _log_int(rng, 16, 32768)  # fewer leave nothing to choose
        case.update(rows=_log_int(rng, 1, max(1, min(256, (1 << 19) // pages))), pages=pages,
                    selected=_log_int(rng, 4, max(4, min(1024, pages // 3))))
        return case
    page = rng.choice([16, 32, 64, 256])
    # scores of pages that are all taken always say nothing
    least = 5 * page if kind == "scores" else 1
    hi = _log_int(rng, max(16, 2 * least), 32768)
    most = {"bounds": 1 << 21, "evict": 1 << 22}.get(kind, 1 << 24)  # keys of all heads
    batch = _log_int(rng, 1, max(1, min(64, most // (hi * kv_heads))))
    lo = max(least, hi - rng.randrange(hi))
    case.update(batch=batch, page_size=page, lo=lo, hi=hi)
    if kind == "bounds":
        case.update(chunk=rng.choice([0, 1, min(lo, _log_int(rng, 1, 2048))]))
    elif kind == "evict":
        budget = _log_int(rng, 8, 16384)
        case.update(budget=budget, first=rng.choice([0, 4, min(budget // 4, 33)]),
                    recent=min(budget // 2, rng.choice([0, 64, 100, 1024])))
    else:
        extent = rng.choice([64, 100, 128, 512, 1000, 1024])
        case.update(rel_extent=extent, window=rng.choice([-1, -1, _log_int(rng, max(64, least), 16384)]))
        if kind == "mass":
            # rows that fit: at most the work of a whole prompt of 16k
            most = max(1, (1 << 33) // (batch * heads * hi))
            case.update(chunk=min(lo, rng.choice([1, _log_int(rng, 1, most), min(most, 4096)])),
                        gathered=rng.random() < 0.5)
        else:
            most = max(1, min(64, (1 << 29) // (batch * heads * hi)))
            case.update(chunk=min(lo, rng.choice([1, 1, _log_int(rng, 1, most)])))
        if kind == "sparse":
            most = (1 << 21) // (batch * case["chunk"] * kv_heads)  # keys of a choice
            case.update(selected=_log_int(rng, 1, max(1, min(8192, most) // page)))
    return case


def _cu(lengths):
    total, out = 0, [0]
    for n in lengths:
        total += n
        out.append(total)
    return out


def _lengths(case):
    """Query and key lengths of a case's sequences (from the case alone)."""
    rng = random.Random(case["shape_seed"])
    lens_k = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    chunk = case.get("chunk", 1)
    return (list(lens_k) if chunk == 0 else [chunk] * case["batch"]), lens_k


def _row_pages(case):
    """How many pages each row of a selection can choose from."""
    rng = random.Random(case["shape_seed"])
    return [rng.randint((case["pages"] + 1) // 2, case["pages"]) for _ in range(case["rows"])]


# --- inputs -----------------------------------------------------------------------------------

def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))

    def randn(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device=dev) * std + mean

    def bf16(*shape, std=1.0, mean=0.0):
        return randn(*shape, std=std, mean=mean).to(torch.bfloat16)

    s = {"case": dict(case)}
    kind, H, K, D = case["kind"], case.get("heads"), case["kv_heads"], HEAD_DIM
    if kind == "select":
        # scores of a page scorer: the first and the last pages of a row are taken always, what is
        # behind its last page never
        T, P = case["rows"], case["pages"]
        n = torch.tensor(_row_pages(case), device=dev)[:, None, None]
        at = torch.arange(P, device=dev)
        x = randn(T, K, P, std=3.0, mean=10.0)
        x = x.masked_fill((at < 1) | (at >= n - 2), math.inf).masked_fill(at >= n, -math.inf)
        s["scores"] = x
        return s

    lens_q, lens_k = _lengths(case)
    B, ps = case["batch"], case["page_size"]
    s["lens_q"], s["lens_k"] = lens_q, lens_k
    s["cu_q"] = torch.tensor(_cu(lens_q), dtype=torch.int32, device=dev)
    s["cu_k"] = torch.tensor(_cu(lens_k), dtype=torch.int32, device=dev)
    T = sum(lens_q)
    # the paged cache: pages in random order
    per_seq = [-(-n // ps) for n in lens_k]
    pages, width = sum(per_seq), max(per_seq)
    perm = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    first = torch.tensor(_cu(per_seq)[:-1], device=dev)[:, None]
    col = torch.arange(width, device=dev)[None, :]
    n_pages = torch.tensor(per_seq, device=dev)[:, None]
    s["table"] = torch.where(col < n_pages, perm[(first + col).clamp(max=pages - 1)],
                             torch.full_like(perm[:1], -1))

    def cache():
        c = torch.empty(pages, ps, K, D, dtype=torch.bfloat16, device=dev)
        step = max(1, 65536 // ps)
        for p in range(0, pages, step):
            c[p:p + step] = bf16(min(step, pages - p), ps, K, D)
        return c

    if kind in ("bounds", "sparse", "mass", "evict"):
        s["k_cache"] = cache()
    if kind in ("sparse", "evict"):
        s["v_cache"] = cache()
    if kind == "bounds":
        s["bounds"] = torch.zeros(pages, K, 2, D, dtype=torch.bfloat16, device=dev)
    if kind == "scores":
        # a page's keys lie around a mean of their own; the extremes of 16 or more of them
        s["bounds"] = torch.empty(pages, K, 2, D, dtype=torch.bfloat16, device=dev)
        for p in range(0, pages, 8192):
            n = min(8192, pages - p)
            mean, spread = randn(n, K, 1, D, std=0.5), randn(n, K, 2, D, std=0.3, mean=1.7).abs()
            s["bounds"][p:p + n] = torch.cat((mean - spread[:, :, :1], mean + spread[:, :, 1:]), dim=2)
    if kind in ("scores", "sparse", "mass"):
        s["q"] = bf16(T, H, D)
        s["rel"] = bf16(T, H, case["rel_extent"], std=0.5)
        s["scale"] = D ** -0.5
    if kind == "sparse":
        # a choice among each row's visible pages, its first and last page always among them
        S = case["selected"]
        b, p = _row_places(s, T)
        last = p[:, None, None] // ps
        at = torch.arange(width, device=dev)
        x = torch.rand(T, K, width, generator=gen, device=dev)
        x = x.masked_fill(at == 0, 2.0).masked_fill(at == last, 3.0).masked_fill(at > last, -1.0)
        S0 = min(S, width)
        val, idx = x.topk(S0, dim=-1)
        idx = torch.where(val >= 0, idx, torch.full_like(idx, width)).sort(dim=-1).values
        idx = torch.where(idx < width, idx, torch.full_like(idx, -1))
        s["pages"] = torch.full((T, K, S), -1, dtype=torch.int32, device=dev)
        s["pages"][:, :, :S0] = idx.to(torch.int32)
    if kind == "mass":
        # the attention's log-sum-exp of unit-variance logits over the visible keys
        b, p = _row_places(s, T)
        seen = p + 1 if case["window"] < 0 else (p + 1).clamp(max=case["window"] + 1)
        s["lse"] = (seen.float().log() + 0.5 + randn(H, T, std=0.1)).contiguous()
        # what earlier steps have gathered; a prompt has no earlier ones
        s["mass"] = randn(B, K, width * ps).abs() if case["gathered"] else None
    if kind == "evict":
        # gathered weights: most keys little, a few very much
        s["mass"] = randn(B, K, width * ps, std=2.0).exp()
    return s


def _row_places(s, total):
    """Sequence and position of every row: queries are the last of their sequence's keys."""
    t = torch.arange(total, device="cuda")
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    b = torch.searchsorted(cu_q, t, right=True) - 1
    shift = (cu_k[1:] - cu_k[:-1]) - (cu_q[1:] - cu_q[:-1])
    return b, t - cu_q[b] + shift[b]


# --- plain forms --------------------------------------------------------------------------------

FIRST_PAGES, LAST_PAGES = 1, 2


def _plain_bounds(s):
    ps, table = s["case"]["page_size"], s["table"].long()
    n_q, n_k = ((s[c][1:] - s[c][:-1]).long()[:, None] for c in ("cu_q", "cu_k"))
    most = max((k - 1) // ps - (k - q) // ps + 1 for q, k in zip(s["lens_q"], s["lens_k"]))
    # the touched pages of each sequence; those behind its last are the last once more
    page = torch.minimum((n_k - n_q) // ps + torch.arange(most, device="cuda"), (n_k - 1) // ps)
    keys = s["k_cache"][table.gather(1, page)].float()
    there = page[..., None] * ps + torch.arange(ps, device="cuda") < n_k[..., None]
    there = there[..., None, None]
    low = keys.masked_fill(~there, math.inf).amin(dim=2)
    high = keys.masked_fill(~there, -math.inf).amax(dim=2)
    s["bounds"][table.gather(1, page)] = torch.stack((low, high), dim=3).to(torch.bfloat16)
    return [s["bounds"]]


def _bias(s, n_keys):
    """Bias [T, H, n_keys] of every key for every row, and which keys the row sees [T, n_keys]."""
    R, W = s["case"]["rel_extent"], s["case"]["window"]
    T, H, _ = s["rel"].shape
    d = _row_places(s, T)[1][:, None] - torch.arange(n_keys, device="cuda")
    bias = s["rel"].float().gather(2, d.clamp(0, R - 1)[:, None, :].expand(T, H, n_keys))
    bias = bias.masked_fill(((d < 0) | (d >= R))[:, None, :], 0.0)
    return bias, (d >= 0) if W < 0 else (d >= 0) & (d <= W)


def _plain_scores(s):
    case = s["case"]
    B, ps, K = case["batch"], case["page_size"], case["kv_heads"]
    T, H, D = s["q"].shape
    P = s["table"].shape[1]
    q = s["q"].float().view(B, T // B, K, H // K, D)
    low, high = s["bounds"][s["table"].clamp(min=0).long()].float().unbind(dim=3)
    x = torch.einsum("btkgd,bpkd->btkgp", q.clamp(min=0.0), high)
    x = x + torch.einsum("btkgd,bpkd->btkgp", q.clamp(max=0.0), low)
    x = (x * s["scale"]).reshape(T, H, P)
    bias, seen = _bias(s, P * ps)
    x = x + bias.masked_fill(~seen[:, None, :], -math.inf).view(T, H, P, ps).amax(dim=-1)
    x = x.view(T, K, H // K, P).amax(dim=2)
    page = seen.view(T, P, ps).any(dim=-1)
    at = torch.arange(P, device="cuda")
    lo = torch.where(page, at, P).amin(dim=1, keepdim=True)
    hi = torch.where(page, at, -1).amax(dim=1, keepdim=True)
    always = page & ((at < lo + FIRST_PAGES) | (at > hi - LAST_PAGES))
    x = x.masked_fill(~page[:, None, :], -math.inf)
    return [x.masked_fill(always[:, None, :], math.inf)]


def _plain_select(s):
    x, S = s["scores"], s["case"]["selected"]
    P = x.shape[-1]
    val, idx = x.sort(dim=-1, descending=True, stable=True)
    val, idx = val[..., :S], idx[..., :S]
    idx = idx.masked_fill(val == -math.inf, P).sort(dim=-1).values
    idx = idx.masked_fill(idx == P, -1).to(torch.int32)
    return [torch.nn.functional.pad(idx, (0, S - idx.shape[-1]), value=-1)]


def _plain_sparse(s):
    case = s["case"]
    ps, K, S, R, W = (case[c] for c in ("page_size", "kv_heads", "selected", "rel_extent", "window"))
    T, H, D = s["q"].shape
    G = H // K
    b, p = _row_places(s, T)
    pages = s["pages"].long()
    place = s["table"].long()[b[:, None, None], pages.clamp(min=0)]
    head = torch.arange(K, device="cuda")[None, :, None]
    k, v = (s[c].permute(0, 2, 1, 3)[place, head].float().view(T, K, S * ps, D)
            for c in ("k_cache", "v_cache"))
    x = torch.einsum("tkgd,tknd->tkgn", s["q"].float().view(T, K, G, D), k) * s["scale"]
    d = p[:, None, None, None] - (pages[..., None] * ps + torch.arange(ps, device="cuda"))
    d = torch.where(pages[..., None] >= 0, d, torch.full_like(d, -1)).view(T, K, 1, S * ps)
    bias = s["rel"].float().view(T, K, G, R).gather(3, d.clamp(0, R - 1).expand(T, K, G, S * ps))
    x = x + bias.masked_fill((d < 0) | (d >= R), 0.0)
    x = x.masked_fill((d < 0) if W < 0 else (d < 0) | (d > W), -math.inf)
    m = x.amax(dim=-1, keepdim=True)
    x = (x - m.masked_fill(m == -math.inf, 0.0)).exp()
    total = x.sum(dim=-1, keepdim=True)
    o = torch.einsum("tkgn,tknd->tkgd", x, v)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return [o.view(T, H, D).to(torch.bfloat16)]


def _plain_mass(s):
    case = s["case"]
    B, ps, K, R, W = (case[c] for c in ("batch", "page_size", "kv_heads", "rel_extent", "window"))
    T, H, D = s["q"].shape
    G, nq, n = H // K, T // B, s["table"].shape[1] * ps
    mass = torch.zeros(B, K, n, device="cuda") if s["mass"] is None else s["mass"]
    k = s["k_cache"][s["table"].clamp(min=0).long()].reshape(B, n, K, D).float()
    p = _row_places(s, T)[1].view(B, nq)
    q, rel = s["q"].view(B, nq, K, G, D), s["rel"].view(B, nq, H, R)
    lse = s["lse"].view(H, B, nq).permute(1, 2, 0)
    step = max(1, (1 << 28) // (B * H * n))  # the logits of all rows at once are too many
    for t in range(0, nq, step):
        at = slice(t, t + step)
        x = torch.einsum("btkgd,bnkd->btkgn", q[:, at].float(), k) * s["scale"]
        x = x.reshape(B, -1, H, n)
        d = (p[:, at, None] - torch.arange(n, device="cuda"))[:, :, None, :]
        bias = rel[:, at].float().gather(3, d.clamp(0, R - 1).expand_as(x))
        x = x + bias.masked_fill((d < 0) | (d >= R), 0.0)
        x = (x - lse[:, at, :, None]).exp()
        x = x.masked_fill((d < 0) if W < 0 else (d < 0) | (d > W), 0.0)
        mass += x.reshape(B, -1, K, G, n).sum(dim=(1, 3))
    return [mass]


def _plain_evict(s):
    case, mass, table = s["case"], s["mass"], s["table"].long()
    ps, budget = case["page_size"], case["budget"]
    B, K, n = mass.shape
    n_k = (s["cu_k"][1:] - s["cu_k"][:-1]).long()[:, None, None]
    at = torch.arange(n, device="cuda")
    always = (at < case["first"]) | (at >= n_k - case["recent"])
    x = mass.masked_fill(always, math.inf).masked_fill(at >= n_k, -math.inf)
    val, idx = x.sort(dim=-1, descending=True, stable=True)
    val, idx = val[..., :budget], idx[..., :budget]
    kept = idx.masked_fill(val == -math.inf, n).sort(dim=-1).values
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=n)
    there = kept < n
    new = n_k.clamp(max=budget)
    # places behind the last kept key repeat it
    to = torch.minimum(torch.arange(budget, device="cuda"), new - 1).expand(B, K, budget)
    source = kept.gather(2, to)
    head = torch.arange(K, device="cuda")[None, :, None]
    seq = torch.arange(B, device="cuda")[:, None, None]
    rows = [s[c][table[seq, source // ps], source % ps, head] for c in ("k_cache", "v_cache")]
    for c, r in zip(("k_cache", "v_cache"), rows):
        s[c][table[seq, to // ps], to % ps, head] = r
    left = torch.nn.functional.pad(mass.gather(2, source), (0, max(0, n - budget)))[..., :n]
    left = left.masked_fill(at >= new, 0.0)
    cu = torch.nn.functional.pad(new.flatten().cumsum(0), (1, 0)).to(torch.int32)
    return [kept.masked_fill(~there, -1).to(torch.int32), left, cu, s["k_cache"], s["v_cache"]]


# --- the package's calls --------------------------------------------------------------------------

def _own(s):
    pkg, case = _package(), s["case"]
    kind = case["kind"]
    if kind == "bounds":
        return [pkg.inkling_kv_page_bounds(s["k_cache"], s["table"], s["cu_q"], s["cu_k"],
                                           max(s["lens_q"]), bounds=s["bounds"])]
    if kind == "select":
        return [pkg.inkling_kv_select_pages(s["scores"], case["selected"])]
    if kind == "evict":
        kept, mass, cu_k = pkg.inkling_kv_evict(
            s["k_cache"], s["v_cache"], s["mass"], s["table"], s["cu_k"], case["budget"],
            first=case["first"], recent=case["recent"])
        return [kept, mass, cu_k, s["k_cache"], s["v_cache"]]
    window = (case["window"], 0)
    if kind == "scores":
        return [pkg.inkling_kv_page_scores(
            s["q"], s["bounds"], s["rel"], s["cu_q"], s["cu_k"], max(s["lens_q"]),
            case["rel_extent"], case["page_size"], window, block_table=s["table"],
            softmax_scale=s["scale"], first_pages=FIRST_PAGES, last_pages=LAST_PAGES)]
    if kind == "sparse":
        return [pkg.inkling_fa4_rel_attention_decode_pages(
            s["q"], s["k_cache"], s["v_cache"], s["rel"], s["cu_q"], s["cu_k"], max(s["lens_q"]),
            max(s["lens_k"]), case["rel_extent"], s["pages"], window, block_table=s["table"],
            softmax_scale=s["scale"])]
    return [pkg.inkling_kv_attention_mass(
        s["q"], s["k_cache"], s["rel"], s["lse"], s["cu_q"], s["cu_k"], max(s["lens_q"]),
        max(s["lens_k"]), case["rel_extent"], window, block_table=s["table"],
        softmax_scale=s["scale"], mass=s["mass"])]


def run(state):
    if own:
        return _own(state)
    plain = {"bounds": _plain_bounds, "scores": _plain_scores, "select": _plain_select,
             "sparse": _plain_sparse, "mass": _plain_mass, "evict": _plain_evict}
    return plain[state["case"]["kind"]](state)


# --- 64 bits, from the definitions ----------------------------------------------------------------

def _largest(x, count):
    """Places of the `count` largest of a vector on the host, the lowest of equal ones first, in
    ascending order; -inf is never among them."""
    order = sorted((i for i, v in enumerate(x) if v != -math.inf), key=lambda i: (-x[i], i))
    return sorted(order[:count])


def _exact_visible(case, s, b, t):
    """Position of row t of sequence b, and the first key it sees."""
    p = s["lens_k"][b] - s["lens_q"][b] + t
    return p, 0 if case["window"] < 0 else max(0, p - case["window"])


def exact(case, seed):
    kind, K = case["kind"], case["kv_heads"]
    if kind == "select" and case["rows"] * K * case["pages"] > 1 << 24:
        return None
    s = prepare(case, seed)
    if kind == "select":
        S = case["selected"]
        picked = [[_largest(row, S) for row in heads] for heads in s["scores"].tolist()]
        return [torch.tensor([[r + [-1] * (S - len(r)) for r in heads] for heads in picked],
                             dtype=torch.int32)]
    B, ps, dev = case["batch"], case["page_size"], "cuda"
    table = s["table"].tolist()

    def rows_of(cache, b, n):
        """Keys or values of the first n places of sequence b, [K, n, D]."""
        pages = torch.tensor(table[b][:-(-n // ps)], device=dev)
        return cache[pages].flatten(0, 1)[:n].transpose(0, 1).double()

    if kind == "bounds":
        out = s["bounds"].double()
        for b, (q, n) in enumerate(zip(s["lens_q"], s["lens_k"])):
            keys = rows_of(s["k_cache"], b, n)
            c0, full = (n - q) // ps, n // ps
            if full > c0:  # whole pages at once, then the one that is not full
                block = keys[:, c0 * ps:full * ps].unflatten(1, (full - c0, ps)).transpose(0, 1)
                at = torch.tensor(table[b][c0:full], device=dev)
                out[at, :, 0], out[at, :, 1] = block.min(2).values, block.max(2).values
            if n % ps:
                tail = keys[:, full * ps:]
                out[table[b][full], :, 0] = tail.min(1).values
                out[table[b][full], :, 1] = tail.max(1).values
        return [out]
    if kind == "evict":
        budget, n_all = case["budget"], s["mass"].shape[-1]
        if B * K * max(s["lens_k"]) > 1 << 23:
            return None
        kept = torch.full((B, K, budget), -1, dtype=torch.int32, device=dev)
        left = torch.zeros(s["mass"].shape, dtype=torch.float64, device=dev)
        caches, cu = [s[c].double() for c in ("k_cache", "v_cache")], [0]
        for b, n in enumerate(s["lens_k"]):
            new = min(n, budget)
            cu.append(cu[-1] + new)
            pages = torch.tensor(table[b], device=dev)
            for g in range(K):
                x = s["mass"][b, g, :n].tolist()
                x = [math.inf if i < case["first"] or i >= n - case["recent"] else v
                     for i, v in enumerate(x)]
                at = torch.tensor(_largest(x, budget), device=dev)
                kept[b, g, :new] = at.to(torch.int32)
                left[b, g, :new] = s["mass"][b, g, at].double()
                to = torch.arange(new, device=dev)
                for cache, name in zip(caches, ("k_cache", "v_cache")):
                    cache[pages[to // ps], to % ps, g] = s[name][pages[at // ps], at % ps, g].double()
        return [kept, left, torch.tensor(cu, dtype=torch.int32, device=dev)] + caches

    H, R = case["heads"], case["rel_extent"]
    G, T = H // K, s["q"].shape[0]
    q = s["q"].double().view(T, K, G, -1)
    rel = s["rel"].double()
    if kind == "scores":
        P = s["table"].shape[1]
        out = torch.full((T, K, P), -math.inf, dtype=torch.float64, device=dev)
        for t in range(T):
            b = t // s["lens_q"][0]
            p, lo = _exact_visible(case, s, b, t % s["lens_q"][0])
            c0, c1 = lo // ps, p // ps + 1
            ends = s["bounds"][torch.tensor(table[b][c0:c1], device=dev)].double()  # [P', K, 2, D]
            far = torch.maximum(q[t][None] * ends[:, :, None, 0], q[t][None] * ends[:, :, None, 1])
            x = far.sum(-1).permute(1, 2, 0) * s["scale"]  # [K, G, P']
            bias = torch.full((H, c1 * ps - c0 * ps), -math.inf, dtype=torch.float64, device=dev)
            bias[:, lo - c0 * ps:p + 1 - c0 * ps] = 0.0
            near = min(p + 1 - lo, R)
            bias[:, p + 1 - near - c0 * ps:p + 1 - c0 * ps] = rel[t, :, :near].flip(1)
            x = x + bias.view(K, G, c1 - c0, ps).max(-1).values
            out[t, :, c0:c1] = x.max(1).values
            out[t, :, c0:min(c1, c0 + FIRST_PAGES)] = math.inf
            out[t, :, max(c0, c1 - LAST_PAGES):c1] = math.inf
        return [out]
    if kind == "sparse":
        out = torch.zeros(T, K, G, HEAD_DIM, dtype=torch.float64, device=dev)
        chosen = s["pages"].tolist()
        if T * K > 4096:
            return None
        for t in range(T):
            b = t // s["lens_q"][0]
            p, lo = _exact_visible(case, s, b, t % s["lens_q"][0])
            for g in range(K):
                mine = [c for c in chosen[t][g] if c >= 0]
                at = (torch.tensor(mine, device=dev)[:, None] * ps
                      + torch.arange(ps, device=dev)).flatten()
                at = at[(at >= lo) & (at <= p)]
                if not at.numel():
                    continue
                pages = s["table"][b].long()[at // ps]
                k, v = (s[c][pages, at % ps, g].double() for c in ("k_cache", "v_cache"))
                d = p - at
                x = q[t, g] @ k.t() * s["scale"]
                x = x + torch.where(d < R, rel[t, g * G:(g + 1) * G, :][:, d.clamp(max=R - 1)], 0.0)
                out[t, g] = x.softmax(-1) @ v
        return [out.view(T, H, HEAD_DIM)]
    # the weights of each head's rows, a stretch of rows at a time
    out, row = torch.zeros(B, K, s["table"].shape[1] * ps, dtype=torch.float64, device=dev), 0
    if s["mass"] is not None:
        out += s["mass"]
    for b, (nq, n) in enumerate(zip(s["lens_q"], s["lens_k"])):
        keys = rows_of(s["k_cache"], b, n)
        step = max(1, (1 << 26) // (G * n))
        for t0 in range(0, nq, step):
            t1 = min(nq, t0 + step)
            seen = n - nq + t1  # keys that these rows can see
            p = torch.arange(n - nq + t0, n - nq + t1, device=dev)
            d = p[:, None] - torch.arange(seen, device=dev)
            gone = (d < 0) | (d > (case["window"] if case["window"] >= 0 else n))
            for g in range(K):
                x = torch.matmul(q[row + t0:row + t1, g], keys[g, :seen].t()) * s["scale"]
                near = (d >= 0) & (d < R)
                r = rel[row + t0:row + t1, g * G:(g + 1) * G].gather(
                    2, d.clamp(0, R - 1)[:, None, :].expand(-1, G, -1))
                x += torch.where(near[:, None, :], r, 0.0)
                x -= s["lse"][g * G:(g + 1) * G, row + t0:row + t1].t()[..., None].double()
                out[b, g, :seen] += torch.where(gone[:, None, :], 0.0, x.exp()).sum(dim=(0, 1))
        row += nq
    return [out]


# --- what a call cannot do without ------------------------------------------------------------------

def work(case):
    K, D = case["kv_heads"], HEAD_DIM
    if case["kind"] == "select":
        n = sum(_row_pages(case)) * K
        return {"bytes": 4 * n + 4 * case["rows"] * K * case["selected"], "flops": n}
    ps, (lens_q, lens_k) = case["page_size"], _lengths(case)
    if case["kind"] == "bounds":
        keys = sum(n - (n - q) // ps * ps for q, n in zip(lens_q, lens_k))
        pages = sum(-(-n // ps) - (n - q) // ps for q, n in zip(lens_q, lens_k))
        return {"bytes": keys * K * D * 2 + pages * K * D * 4, "flops": 2 * keys * K * D}
    if case["kind"] == "evict":
        # which keys stay is known with the masses only: every kept one but the first moves
        rows = sum(min(n, case["budget"]) for n in lens_k if n > case["budget"])
        return {"bytes": (sum(lens_k) * 8 + rows * D * 8 + case["batch"] * case["budget"] * 4) * K,
                "flops": sum(lens_k) * K}
    H, R, W = case["heads"], case["rel_extent"], case["window"]
    T = sum(lens_q)
    # visible keys of each row (all the rows of a sequence end at its last keys)
    seen = [[min(p + 1, W + 1) if W >= 0 else p + 1 for p in range(n - q, n)]
            for q, n in zip(lens_q, lens_k)]
    total = sum(map(sum, seen))
    rel = sum(min(x, R) for row in seen for x in row) * H * 2
    rows_bytes = T * H * D * 2
    if case["kind"] == "scores":
        pages = [[(n - q + t) // ps - (n - q + t + 1 - x) // ps + 1 for t, x in enumerate(row)]
                 for q, n, row in zip(lens_q, lens_k, seen)]
        width = max(-(-n // ps) for n in lens_k)
        read = sum((n - 1) // ps - (n - q + 1 - row[0]) // ps + 1
                   for q, n, row in zip(lens_q, lens_k, seen))
        return {"bytes": read * K * D * 4 + T * K * width * 4 + rows_bytes + rel,
                "flops": 4 * D * H * sum(map(sum, pages))}
    if case["kind"] == "sparse":
        keys = sum(min(x, case["selected"] * ps) for row in seen for x in row)
        return {"bytes": keys * K * D * 4 + rows_bytes * 2 + T * K * case["selected"] * 4
                + sum(min(x, R, case["selected"] * ps) for row in seen for x in row) * H * 2,
                "flops": 4 * D * H * keys}
    keys = sum(min(n, n - (n - q + 1 - row[0])) for q, n, row in zip(lens_q, lens_k, seen))
    return {"bytes": keys * K * (D * 2 + 8) + rows_bytes + rel + T * H * 4,
            "flops": 2 * D * H * total}
