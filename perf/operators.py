"""The operators next to the relative-bias attention, in their plain form and as the package's
calls, over the sizes they meet: the norm and rotation of queries and keys in front of the
attention (forward and gradients), the append of new keys and values to the paged cache, decode
for a batch whose sequences share a prefix, and the learned bias by distance buckets with its
gradient.

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
EPS = 1e-6
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
        # one short sequence, few heads: the smallest training or prefill call (latency)
        {"name": "norm_rope_s128", "kind": "norm_rope", "tokens": 128, "seqs": 1, "heads": 4,
         "kv_heads": 4, "rotary_dim": 128, "interleaved": False, "weights": "bf16", "grad": False,
         "past": 0, "shape_seed": 0},
        # a ragged prefill batch, partial rotation of neighbouring pairs
        {"name": "norm_rope_ragged16", "kind": "norm_rope", "tokens": 30011, "seqs": 16,
         "heads": 32, "kv_heads": 8, "rotary_dim": 64, "interleaved": True, "weights": "bf16",
         "grad": False, "past": 0, "shape_seed": 1},
        # the forward and the gradients of one long training sequence
        {"name": "norm_rope_train_32k", "kind": "norm_rope", "tokens": 32768, "seqs": 1,
         "heads": 32, "kv_heads": 8, "rotary_dim": 128, "interleaved": False, "weights": "fp32",
         "grad": True, "past": 0, "shape_seed": 2},
        # one sequence generating one token (latency)
        {"name": "append_decode_b1", "kind": "append", "batch": 1, "chunk": 1, "lo": 4096,
         "hi": 4096, "heads": 32, "kv_heads": 8, "page_size": 16, "rotary_dim": 128,
         "interleaved": False, "shape_seed": 3},
        # a decode batch: one token for each of 128 sequences
        {"name": "append_decode_b128", "kind": "append", "batch": 128, "chunk": 1, "lo": 256,
         "hi": 2048, "heads": 32, "kv_heads": 8, "page_size": 16, "rotary_dim": 128,
         "interleaved": False, "shape_seed": 4},
        # chunked prefill: 8 chunks of 2048 tokens behind 16384 cached ones
        {"name": "append_chunks_8x2048", "kind": "append", "batch": 8, "chunk": 2048,
         "lo": 18432, "hi": 18432, "heads": 32, "kv_heads": 8, "page_size": 64,
         "rotary_dim": 64, "interleaved": False, "shape_seed": 5},
        # a few sequences behind a short common prompt (latency)
        {"name": "prefix_b8_2k", "kind": "prefix", "batch": 8, "prefix": 2048, "lo": 1, "hi": 128,
         "heads": 32, "kv_heads": 8, "rel_extent": 128, "page_size": 16, "window": -1,
         "shape_seed": 6},
        # an odd batch, a head group of three, a long bias and an odd number of pages
        {"name": "prefix_b33_10k_g3", "kind": "prefix", "batch": 33, "prefix": 10032, "lo": 1,
         "hi": 700, "heads": 12, "kv_heads": 4, "rel_extent": 1000, "page_size": 16,
         "window": -1, "shape_seed": 7},
        # a large decode batch behind one long document
        {"name": "prefix_b128_32k", "kind": "prefix", "batch": 128, "prefix": 32768, "lo": 1,
         "hi": 1024, "heads": 32, "kv_heads": 8, "rel_extent": 128, "page_size": 64,
         "window": -1, "shape_seed": 8},
        # the bias table of one short sequence and its gradient (latency)
        {"name": "bucket_bias_s128", "kind": "bucket", "tokens": 128, "heads": 4,
         "rel_extent": 128, "buckets": 32, "max_distance": 128, "weights": "fp32",
         "shape_seed": 9},
        # the layers with a short bias over one long training sequence
        {"name": "bucket_bias_32k_r128", "kind": "bucket", "tokens": 32768, "heads": 32,
         "rel_extent": 128, "buckets": 32, "max_distance": 128, "weights": "bf16",
         "shape_seed": 10},
        # the layers with the longest bias; logarithmic buckets far beyond the exact ones
        {"name": "bucket_bias_32k_r1024", "kind": "bucket", "tokens": 32768, "heads": 32,
         "rel_extent": 1024, "buckets": 64, "max_distance": 1024, "weights": "fp32",
         "shape_seed": 11},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_rope", "append", "prefix", "bucket"])
    heads, kv_heads = rng.choice([(4, 4), (8, 2), (12, 4), (32, 8), (16, 16), (5, 1)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads,
            "shape_seed": rng.randrange(1 << 20)}
    if kind == "norm_rope":
        tokens = _log_int(rng, 1, 32768)
        case.update(tokens=tokens, seqs=min(tokens, _log_int(rng, 1, 64)),
                    rotary_dim=rng.choice([0, 32, 64, 96, 128]),
                    interleaved=rng.random() < 0.5, weights=rng.choice(["bf16", "fp32", "none"]),
                    grad=rng.random() < 0.5, past=rng.choice([0, 0, 7, 100000]))
    elif kind == "append":
        batch = _log_int(rng, 1, 256)
        chunk = _log_int(rng, 1, max(1, 16384 // batch))
        lo = chunk + _log_int(rng, 1, max(1, 65536 // batch))
        case.update(batch=batch, chunk=chunk, lo=lo, hi=lo + rng.randrange(300),
                    page_size=rng.choice([16, 32, 64, 256]),
                    rotary_dim=rng.choice([0, 32, 64, 128]), interleaved=rng.random() < 0.5)
    elif kind == "prefix":
        batch = _log_int(rng, 2, 128)
        page = rng.choice([16, 32, 64, 128])
        lo = rng.choice([0, 1, 1, 40])
        case.update(batch=batch, page_size=page, prefix=page * max(1, _log_int(rng, 16, 32768) // page),
                    lo=lo, hi=lo + _log_int(rng, 1, 1024),
                    rel_extent=rng.choice([64, 100, 128, 512, 1000, 1024]),
                    window=rng.choice([-1, -1, _log_int(rng, 64, 16384)]))
    else:
        extent = rng.choice([64, 100, 128, 200, 512, 1000, 1024])
        buckets = rng.choice([8, 20, 32, 64, 128])
        case.update(tokens=_log_int(rng, 1, 32768), rel_extent=extent, buckets=buckets,
                    max_distance=max(buckets, rng.choice([64, 128, 500, 1024])),
                    weights=rng.choice(["bf16", "fp32"]))
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
    if case["kind"] == "norm_rope":
        cuts = sorted(rng.sample(range(1, case["tokens"]), case["seqs"] - 1))
        lens = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
        return lens, [n + case["past"] for n in lens]
    n = case["batch"]
    own_keys = [rng.randint(case["lo"], case["hi"]) for _ in range(n)]
    if case["kind"] == "append":
        return [case["chunk"]] * n, own_keys
    return [1] * n, [case["prefix"] + s for s in own_keys]


def bucket_starts(buckets, max_distance):
    """First distance of each bucket: half of them hold one distance each, the others grow
    logarithmically up to max_distance (bucket b >= e starts at the first d with
    (d / e)^(buckets - e) >= (max_distance / e)^(b - e), in whole numbers)."""
    e = buckets // 2
    n = buckets - e
    starts, d = list(range(e)), e
    for j in range(n):
        want = max_distance ** j * e ** (n - j)
        while d ** n < want:
            d += 1
        starts.append(d)
    return starts


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
    H, K, D = case["heads"], case.get("kv_heads"), HEAD_DIM
    if case["kind"] == "bucket":
        T, R, B = case["tokens"], case["rel_extent"], case["buckets"]
        wt = torch.bfloat16 if case["weights"] == "bf16" else torch.float32
        s["table"] = randn(B, H, std=0.5).to(wt)
        s["starts"] = torch.tensor(bucket_starts(B, case["max_distance"]), dtype=torch.int32,
                                   device=dev)
        # the attention's gradients of its logits: small, of both signs
        s["drel"] = torch.empty(T, H, R, dtype=torch.bfloat16, device=dev)
        for t in range(0, T, 4096):
            n = min(4096, T - t)
            s["drel"][t:t + n] = bf16(n, H, R, std=0.01)
        return s

    lens_q, lens_k = _lengths(case)
    s["lens_q"], s["lens_k"] = lens_q, lens_k
    s["cu_q"] = torch.tensor(_cu(lens_q), dtype=torch.int32, device=dev)
    s["cu_k"] = torch.tensor(_cu(lens_k), dtype=torch.int32, device=dev)
    T = sum(lens_q)
    if case["kind"] in ("norm_rope", "append"):
        # q, k, v are slices of one projection's output, as a layer has them
        merged = bf16(T, (H + 2 * K) * D)
        s["q"] = merged[:, :H * D].view(T, H, D)
        s["k"] = merged[:, H * D:(H + K) * D].view(T, K, D)
        s["v"] = merged[:, (H + K) * D:].view(T, K, D)
        weights = case.get("weights", "bf16")
        s["wq"] = s["wk"] = None
        if weights != "none":
            wt = torch.bfloat16 if weights == "bf16" else torch.float32
            s["wq"], s["wk"] = (randn(D, std=0.2, mean=1.0).to(wt) for _ in range(2))
        rot = case["rotary_dim"]
        s["inv_freq"] = None
        if rot:
            s["inv_freq"] = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot).to(dev)
        if case.get("grad"):
            s["dq"], s["dk"] = bf16(T, H, D, std=0.1), bf16(T, K, D, std=0.1)
    if case["kind"] == "norm_rope":
        return s

    # the paged cache: pages in random order; the sequences of a prefix case begin with the same
    ps = case["page_size"]
    shared = case.get("prefix", 0) // ps
    own_pages = [-(-n // ps) - shared for n in lens_k]
    pages = shared + sum(own_pages)
    perm = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    width = shared + max(own_pages)
    own_first = torch.tensor(_cu(own_pages)[:-1], device=dev)[:, None] + shared
    col = torch.arange(width, device=dev)[None, :]
    at = torch.where(col < shared, col.expand(len(lens_k), width), own_first + col - shared)
    n_pages = torch.tensor(own_pages, device=dev)[:, None] + shared
    s["table"] = torch.where(col < n_pages, perm[at.clamp(max=pages - 1)], torch.full_like(perm[:1], -1))
    s["k_cache"], s["v_cache"] = (torch.empty(pages, ps, K, D, dtype=torch.bfloat16, device=dev)
                                  for _ in range(2))
    step = max(1, 65536 // ps)
    for c in (s["k_cache"], s["v_cache"]):
        for p in range(0, pages, step):
            n = min(step, pages - p)
            c[p:p + n] = bf16(n, ps, K, D)
    if case["kind"] == "prefix":
        s["q"] = bf16(T, H, D)
        s["rel"] = bf16(T, H, case["rel_extent"], std=0.5)
        s["scale"] = D ** -0.5
    return s


# --- plain forms --------------------------------------------------------------------------------

def _positions(s, total):
    """Sequence and position of every token: queries are the last of their sequence's keys."""
    t = torch.arange(total, device="cuda")
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    b = torch.searchsorted(cu_q, t, right=True) - 1
    shift = (cu_k[1:] - cu_k[:-1]) - (cu_q[1:] - cu_q[:-1])
    return b, t - cu_q[b] + shift[b]


def _cos_sin(s, total):
    # angles of far positions need 64 bits
    angle = _positions(s, total)[1].double()[:, None] * s["inv_freq"]
    return angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]


def _halves(x, rot, interleaved):
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _join(a, b, rest, interleaved):
    both = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((both, rest), dim=-1)


def _rotate(x, cos, sin, rot, interleaved):
    a, b = _halves(x, rot, interleaved)
    return _join(a * cos - b * sin, a * sin + b * cos, x[..., rot:], interleaved)


def _norm_rope(s, x, w):
    case = s["case"]
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(dim=-1, keepdim=True) + EPS)
    if w is not None:
        y = y * w.float()
    if case["rotary_dim"]:
        y = _rotate(y, *_cos_sin(s, x.shape[0]), case["rotary_dim"], case["interleaved"])
    return y.to(torch.bfloat16)


def _norm_rope_grad(s, dy, x, w):
    case = s["case"]
    g = dy.float()
    if case["rotary_dim"]:
        cos, sin = _cos_sin(s, x.shape[0])
        g = _rotate(g, cos, -sin, case["rotary_dim"], case["interleaved"])
    xf = x.float()
    r = torch.rsqrt((xf * xf).mean(dim=-1, keepdim=True) + EPS)
    xhat = xf * r
    dw = None if w is None else (g * xhat).sum(dim=(0, 1)).to(w.dtype)
    if w is not None:
        g = g * w.float()
    dx = (g - xhat * (g * xhat).mean(dim=-1, keepdim=True)) * r
    return dx.to(torch.bfloat16), dw


def _plain_norm_rope(s):
    out = [_norm_rope(s, s["q"], s["wq"]), _norm_rope(s, s["k"], s["wk"])]
    if s["case"]["grad"]:
        dq, dwq = _norm_rope_grad(s, s["dq"], s["q"], s["wq"])
        dk, dwk = _norm_rope_grad(s, s["dk"], s["k"], s["wk"])
        out += [dq, dk, dwq, dwk]
    return out


def _plain_append(s):
    b, pos = _positions(s, s["k"].shape[0])
    ps = s["case"]["page_size"]
    page, slot = s["table"][b, pos // ps].long(), pos % ps
    s["k_cache"][page, slot] = _norm_rope(s, s["k"], s["wk"])
    s["v_cache"][page, slot] = s["v"]
    return [_norm_rope(s, s["q"], s["wq"]), s["k_cache"], s["v_cache"]]


def _plain_prefix(s):
    case = s["case"]
    P, ps, K, R = case["prefix"], case["page_size"], case["kv_heads"], case["rel_extent"]
    B, H, D = s["q"].shape
    n_keys = (s["cu_k"][1:] - s["cu_k"][:-1]).long()
    first = P // ps
    q = s["q"].float().view(B, K, H // K, D)

    def logits(keys, k_pos):
        x = torch.einsum("bkgd,pkd->bkgp" if keys.dim() == 3 else "bkgd,bpkd->bkgp", q, keys)
        x = x * s["scale"]
        d = n_keys[:, None] - 1 - k_pos[None, :]
        bias = s["rel"].float().gather(2, d.clamp(0, R - 1)[:, None, :].expand(B, H, -1))
        near = ((d >= 0) & (d < R))[:, None, None, :]
        x = x + torch.where(near, bias.view(B, K, H // K, -1), torch.zeros_like(x))
        seen = (d >= 0) if case["window"] < 0 else (d >= 0) & (d <= case["window"])
        return x.masked_fill(~seen[:, None, None, :], -math.inf)

    shared = s["table"][0, :first].long()
    kp, vp = (s[c][shared].reshape(P, K, D).float() for c in ("k_cache", "v_cache"))
    tail = s["table"][:, first:].clamp(min=0).long()
    n = tail.shape[1] * ps
    ks, vs = (s[c][tail].reshape(B, n, K, D).float() for c in ("k_cache", "v_cache"))
    a = logits(kp, torch.arange(P, device="cuda"))
    c = logits(ks, P + torch.arange(n, device="cuda"))
    m = torch.maximum(a.amax(-1, keepdim=True), c.amax(-1, keepdim=True)) if n else a.amax(-1, keepdim=True)
    m = m.masked_fill(m == -math.inf, 0.0)
    a, c = (a - m).exp(), (c - m).exp()
    total = a.sum(-1, keepdim=True) + c.sum(-1, keepdim=True)
    o = torch.einsum("bkgp,pkd->bkgd", a, vp) + torch.einsum("bkgp,bpkd->bkgd", c, vs)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return [o.view(B, H, D).to(torch.bfloat16)]


def _plain_bucket(s):
    T, H, R = s["drel"].shape
    table = s["table"]
    bucket = torch.searchsorted(s["starts"], torch.arange(R, device="cuda", dtype=torch.int32),
                                right=True) - 1
    rel = table.float()[bucket].t().to(torch.bfloat16)
    sums = s["drel"].sum(dim=0, dtype=torch.float32)
    grad = torch.zeros(table.shape, device="cuda").index_add(0, bucket, sums.t())
    return [rel.unsqueeze(0).expand(T, H, R), grad.to(table.dtype)]


# --- the package's calls --------------------------------------------------------------------------

def _own(s):
    pkg, case = _package(), s["case"]
    kind = case["kind"]
    if kind == "norm_rope":
        rope = {"inv_freq": s["inv_freq"], "interleaved": case["interleaved"], "eps": EPS}
        out = list(pkg.inkling_qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cu_q"],
                                            s["cu_k"], **rope))
        if case["grad"]:
            out += pkg.inkling_qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["wq"],
                                                     s["wk"], s["cu_q"], s["cu_k"], **rope)
        return out
    if kind == "append":
        q = pkg.inkling_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"],
                                  s["cu_q"], s["cu_k"], q=s["q"], q_weight=s["wq"],
                                  k_weight=s["wk"], eps=EPS, inv_freq=s["inv_freq"],
                                  interleaved=case["interleaved"])
        return [q, s["k_cache"], s["v_cache"]]
    if kind == "prefix":
        return [pkg.inkling_fa4_rel_attention_decode_shared_prefix(
            s["q"], s["k_cache"], s["v_cache"], s["rel"], s["cu_q"], s["cu_k"], 1,
            max(s["lens_k"]), case["rel_extent"], case["prefix"],
            window_size=(case["window"], 0), softmax_scale=s["scale"],
            block_table=s["table"])]
    rel = pkg.inkling_bucket_bias(s["table"], s["starts"], s["drel"].shape[0],
                                  case["rel_extent"])
    return [rel, pkg.inkling_bucket_bias_backward(s["drel"], s["starts"], case["buckets"],
                                                  dtype=s["table"].dtype)]


def run(state):
    if own:
        return _own(state)
    plain = {"norm_rope": _plain_norm_rope, "append": _plain_append, "prefix": _plain_prefix,
             "bucket": _plain_bucket}
    return plain[state["case"]["kind"]](state)


# --- 64 bits, from the definitions ----------------------------------------------------------------

def _exact_rows(s, x, w):
    """Unit root mean square, scaled, then each pair turned as a complex number."""
    case = s["case"]
    y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
    if w is not None:
        y = y * w
    rot = case["rotary_dim"]
    if not rot:
        return y
    pos = torch.cat([torch.arange(nk - nq, nk, device="cuda") for nq, nk in
                     zip(s["lens_q"], s["lens_k"])]).double()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       pos[:, None, None] * s["inv_freq"])
    head = y[..., :rot]
    pairs = head.unflatten(-1, (rot // 2, 2) if case["interleaved"] else (2, rot // 2))
    if not case["interleaved"]:
        pairs = pairs.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    if not case["interleaved"]:
        z = z.transpose(-1, -2)
    return torch.cat((z.flatten(-2), y[..., rot:]), dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm_rope":
        outs, grads, dws = [], [], []
        for x, w, g in ((s["q"], s["wq"], s.get("dq")), (s["k"], s["wk"], s.get("dk"))):
            x = x.double().requires_grad_(case["grad"])
            w = w if w is None else w.double().requires_grad_(case["grad"])
            y = _exact_rows(s, x, w)
            if case["grad"]:
                got = torch.autograd.grad(y, [x] if w is None else [x, w], g.double())
                grads.append(got[0])
                dws.append(got[1] if w is not None else None)
            outs.append(y.detach())
        return outs + grads + dws
    if case["kind"] == "append":
        caches = [s[c].double() for c in ("k_cache", "v_cache")]
        new = (_exact_rows(s, s["k"].double(), s["wk"].double()), s["v"].double())
        ps, t = case["page_size"], 0
        for b, (nq, nk) in enumerate(zip(s["lens_q"], s["lens_k"])):
            at = torch.arange(nk - nq, nk, device="cuda")
            flat = s["table"][b].long()[at // ps] * ps + at % ps
            for cache, rows in zip(caches, new):
                cache.view(-1, *cache.shape[2:])[flat] = rows[t:t + nq]
            t += nq
        return [_exact_rows(s, s["q"].double(), s["wq"].double())] + caches
    if case["kind"] == "prefix":
        H, K, R = case["heads"], case["kv_heads"], case["rel_extent"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens_k"]):
            pages = s["table"][b, :-(-n // case["page_size"])].long()
            k, v = (s[c][pages].flatten(0, 1)[:n].double().repeat_interleave(H // K, dim=1)
                    for c in ("k_cache", "v_cache"))
            x = (k * s["q"][b].double()).sum(-1).t() * s["scale"]
            near = min(n, R)
            x[:, n - near:] += s["rel"][b, :, :near].double().flip(1)
            if case["window"] >= 0:
                x[:, :max(0, n - 1 - case["window"])] = -math.inf
            out[b] = (x.softmax(-1).t().unsqueeze(-1) * v).sum(0)
        return [out]
    T, H, R = s["drel"].shape
    starts = bucket_starts(case["buckets"], case["max_distance"]) + [R]
    rel = torch.empty(H, R, dtype=torch.float64, device="cuda")
    grad = torch.zeros(case["buckets"], H, dtype=torch.float64, device="cuda")
    for i, (a, b) in enumerate(zip(starts[:-1], starts[1:])):
        a, b = min(a, R), min(b, R)
        rel[:, a:b] = s["table"][i].double()[:, None]
        grad[i] = s["drel"][:, :, a:b].sum(dim=(0, 2), dtype=torch.float64)
    return [rel.expand(T, H, R), grad]


# --- what a call cannot do without ------------------------------------------------------------------

def work(case):
    H, K, D = case["heads"], case.get("kv_heads"), HEAD_DIM
    if case["kind"] == "bucket":
        T, R, B = case["tokens"], case["rel_extent"], case["buckets"]
        size = 2 if case["weights"] == "bf16" else 4
        return {"bytes": T * H * R * 2 + H * R * 2 + 2 * B * H * size + 4 * B, "flops": T * H * R}
    lens_q, lens_k = _lengths(case)
    T = sum(lens_q)
    if case["kind"] == "norm_rope":
        row = (H + K) * D * 2
        return {"bytes": T * row * (5 if case["grad"] else 2),
                "flops": T * (H + K) * D * (30 if case["grad"] else 10)}
    if case["kind"] == "append":
        return {"bytes": T * (H + 2 * K) * D * 2 * 2, "flops": T * (H + K) * D * 10}
    P, R, W = case["prefix"], case["rel_extent"], case["window"]
    seen = [n if W < 0 else min(n, W + 1) for n in lens_k]
    prefix = max(max(0, m - (n - P)) for m, n in zip(seen, lens_k))
    keys = prefix + sum(min(m, n - P) for m, n in zip(seen, lens_k))
    return {"bytes": keys * K * D * 4 + T * H * D * 4 + sum(min(m, R) for m in seen) * H * 2,
            "flops": 4 * D * H * sum(seen)}
