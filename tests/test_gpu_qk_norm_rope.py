"""Norm and rotation of query and key heads on the GPU, its gradients, and the append to the paged
cache, against the 64-bit oracle (oracle/operators_oracle.py).

Tolerances.  A value rounded to bf16 is off by at most 2^-8 of itself.  Before that rounding the
fp32 work on a value y in a rotated pair of length s makes errors relative to s: the mean of 128
squares (7 register and 4 shuffle additions, at most 12 roundings, halved by the root), rsqrt
(2 ulp), eps and two multiplications, cosine and sine (2 ulp each, and 2e-7 = 3.4 * 2^-24 of angle),
two products and an addition: under 32 roundings of 2^-24, so 2^-19 s.  The gradient dx adds the dot
product (another 12 roundings) and three products: 2^-18 of the sizes of its two terms.  A weight
gradient is a sum of terms off by 2^-18 each, added along at most 256 additions (32 a lane at these
sizes, 8 half-warps, 28 blocks a thread, 32 threads): (2^-18 + 256 * 2^-24) of the sum of sizes."""
import numpy as np
import pytest
import torch

import oracle
from gpu_util import device_status_ok
from inkling_fa4 import (_ops, inkling_kv_append, inkling_qk_norm_rope,
                         inkling_qk_norm_rope_backward)
from inkling_fa4.workloads import cu_from_lens

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert device_status_ok(), "a kernel abandoned a bounded wait"


@pytest.fixture(params=[True, False], ids=["ops", "ctypes"])
def both_paths(request):
    before = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = request.param
    yield
    _ops.USE_TORCH_OPS = before


def _randn(*shape, seed, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(*shape, generator=g)).to(dtype)


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _inv_freq(rot, theta=10000.0, dtype=torch.float64):
    if rot == 0:
        return None
    return (theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).to(dtype)


def _weights(kind, seed=9):
    if kind is None:
        return None, None
    return tuple((1 + _randn(128, seed=seed + i, std=0.3, dtype=torch.float32)).to(kind)
                 for i in range(2))


def _dev(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _check_rows(got, want, inv, interleaved, what=""):
    size = oracle.norm_rope_pair_size(want, inv, interleaved)
    err = np.abs(_np(got) - want) - (2.0 ** -8 * np.abs(want) + 2.0 ** -19 * size + 1e-30)
    assert err.max() <= 0, f"{what}: {err.max()}"


CASES = [  # lens_q, lens_k (None: no cu_k; both None: no cu_q), heads, kv, rot, interleaved, w, eps
    (([7], None), 4, 4, 128, False, torch.bfloat16, 1e-6),
    (([1], [100000000]), 5, 1, 128, False, torch.float32, 1e-6),
    (([130, 0, 1, 33], [130, 5, 9000, 40]), 8, 2, 64, True, torch.bfloat16, 1e-5),
    (([300, 17], None), 12, 4, 96, False, torch.float32, 1e-6),
    (([257], None), 3, 3, 32, True, None, 1e-6),
    (([64, 64], [64, 100]), 32, 8, 16, False, torch.bfloat16, 0.0),
    (([100], None), 4, 1, 0, False, torch.bfloat16, 1e-6),
    (([100, 3], None), 4, 2, 128, True, None, None),
    ((list(range(70)), None), 6, 2, 128, False, torch.float32, 1e-6),
    (([5], [2]), 4, 4, 64, False, torch.bfloat16, 1e-6),     # fewer keys than queries
]


@pytest.mark.parametrize("lens,heads,kv,rot,inter,wt,eps", CASES)
def test_forward_and_gradients(lens, heads, kv, rot, inter, wt, eps):
    lens_q, lens_k = lens
    T = sum(lens_q)
    cu_q = cu_from_lens(lens_q)
    cu_k = None if lens_k is None else cu_from_lens(lens_k)
    q, k = _randn(T, heads, 128, seed=1), _randn(T, kv, 128, seed=2, std=3.0)
    gq, gk = _randn(T, heads, 128, seed=3), _randn(T, kv, 128, seed=4, std=0.01)
    wq, wk = _weights(wt)
    inv = _inv_freq(rot)
    pos = oracle.token_positions(T, cu_q.numpy(), None if cu_k is None else cu_k.numpy())
    dev = _dev(q, k, wq, wk, cu_q, cu_k)
    kw = dict(eps=eps, inv_freq=None if inv is None else inv.cuda(), interleaved=inter)
    outs = inkling_qk_norm_rope(*dev, **kw)
    grads = inkling_qk_norm_rope_backward(gq.cuda(), gk.cuda(), *dev, **kw)
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        want = oracle.norm_rope(_np(x), _np(w), pos, eps, _np(inv), inter)
        _check_rows(outs[i], want, _np(inv), inter, f"output {i}")
        dx, dw, dx_size, dw_size = oracle.norm_rope_grads(_np(g), _np(x), _np(w), pos, eps,
                                                          _np(inv), inter)
        err = np.abs(_np(grads[i]) - dx) - (2.0 ** -8 * np.abs(dx) + 2.0 ** -18 * dx_size)
        assert err.max() <= 0, f"gradient {i}: {err.max()}"
        if w is None:
            assert grads[2 + i] is None
            continue
        assert grads[2 + i].dtype == w.dtype
        tol = (2.0 ** -18 + 256 * 2.0 ** -24) * dw_size
        if w.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * (np.abs(dw) + tol)
        assert (np.abs(_np(grads[2 + i]) - dw) <= tol).all(), f"weight gradient {i}"


def test_no_sequences_given_means_one(both_paths):
    q, k = _randn(50, 4, 128, seed=1), _randn(50, 2, 128, seed=2)
    inv = _inv_freq(128, dtype=torch.float32)
    got = inkling_qk_norm_rope(q.cuda(), k.cuda(), inv_freq=inv.cuda())
    for g, x in zip(got, (q, k)):
        want = oracle.norm_rope(_np(x), None, np.arange(50), 1e-6, _np(inv), False)
        _check_rows(g, want, _np(inv), False)


def test_far_positions_keep_their_angles():
    """Positions near 2^31 with frequencies up to 3: the angle in 64 bits on the CPU is itself
    good to 2^31 * 3 * 2^-53 = 7e-7, added to the tolerance relative to the pair."""
    T = 9
    q = _randn(T, 2, 128, seed=5)
    inv = torch.linspace(1e-9, 3.0, 64, dtype=torch.float64)
    cu_q, cu_k = cu_from_lens([T]), torch.tensor([0, 2 ** 31 - 1], dtype=torch.int32)
    got, _ = inkling_qk_norm_rope(*_dev(q, q, None, None, cu_q, cu_k), inv_freq=inv.cuda())
    pos = oracle.token_positions(T, cu_q.numpy(), cu_k.numpy())
    want = oracle.norm_rope(_np(q), None, pos, 1e-6, _np(inv), False)
    size = oracle.norm_rope_pair_size(want, _np(inv), False)
    err = np.abs(_np(got) - want) - (2.0 ** -8 * np.abs(want) + (2.0 ** -19 + 1.5e-6) * size)
    assert err.max() <= 0


@pytest.mark.parametrize("values", ["zero", "huge", "tiny"])
def test_extreme_rows(values):
    """Rows of zeros (eps keeps them 0), of 1e18 (their squares still sum in fp32) and of 1e-30
    (below eps)."""
    x = {"zero": torch.zeros(4, 2, 128), "huge": 1e18 * torch.ones(4, 2, 128),
         "tiny": 1e-30 * torch.ones(4, 2, 128)}[values].to(torch.bfloat16)
    got, _ = inkling_qk_norm_rope(x.cuda(), x.cuda())
    want = oracle.norm_rope(_np(x), None, np.arange(4), 1e-6, None, False)
    _check_rows(got, want, None, False)


def test_nan_and_inf_stay_in_their_rows():
    x = _randn(6, 3, 128, seed=8)
    bad = x.clone()
    bad[2, 1, 5], bad[4, 0, 100] = float("nan"), float("inf")
    inv = _inv_freq(64).cuda()
    a, b = (inkling_qk_norm_rope(t.cuda(), t.cuda(), inv_freq=inv)[0] for t in (x, bad))
    mask = torch.ones(6, 3, dtype=torch.bool)
    mask[2, 1] = mask[4, 0] = False
    assert torch.equal(a[mask.cuda()], b[mask.cuda()])
    assert bool(torch.isnan(b[2, 1].float()).any()) and bool(torch.isnan(b[4, 0].float()).any())
    # without the norm an infinity outside the rotated dims stays what it is
    c, _ = inkling_qk_norm_rope(bad.cuda(), bad.cuda(), eps=None, inv_freq=inv)
    assert torch.equal(c[4, 0, 64:].cpu(), bad[4, 0, 64:])


def test_strided_inputs_and_rows_behind_the_last_sequence(both_paths):
    T, H, K = 40, 6, 2
    merged = _randn(T, (H + 2 * K) * 128 + 8, seed=6)
    cu = cu_from_lens([20, 9])  # rows 29.. are padding
    m = merged.cuda()
    q, k = m[:, :H * 128].view(T, H, 128), m[:, H * 128:(H + K) * 128].view(T, K, 128)
    wq, wk = _dev(*_weights(torch.float32))
    inv = _inv_freq(128).cuda()
    qo, ko = inkling_qk_norm_rope(q, k, wq, wk, cu.cuda(), inv_freq=inv)
    want = inkling_qk_norm_rope(q.contiguous(), k.contiguous(), wq, wk, cu.cuda(), inv_freq=inv)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    assert bool((qo[29:] == 0).all()) and bool((ko[29:] == 0).all())
    g = torch.full_like(qo, float("nan"))
    g[:29] = 1.0
    gk = torch.ones_like(ko)
    dq, dk, dwq, dwk = inkling_qk_norm_rope_backward(g, gk, q, k, wq, wk, cu.cuda(), inv_freq=inv)
    assert bool((dq[29:] == 0).all()) and bool((dk[29:] == 0).all())
    assert bool(torch.isfinite(dwq).all()) and bool(torch.isfinite(dq.float()).all())
    d2 = inkling_qk_norm_rope_backward(g[:29].contiguous(), gk[:29].contiguous(), q[:29], k[:29],
                                       wq, wk, cu.cuda(), inv_freq=inv)
    assert torch.equal(dq[:29], d2[0])
    # a last dimension that is not contiguous, an odd offset and a broadcast row are copied
    odd = m[:, 1:1 + H * 128].view(T, H, 128)
    assert torch.equal(inkling_qk_norm_rope(odd, k, inv_freq=inv)[0],
                       inkling_qk_norm_rope(odd.contiguous(), k, inv_freq=inv)[0])
    tr = m[:, :H * 128].view(T, 128, H).transpose(1, 2)
    assert torch.equal(inkling_qk_norm_rope(tr, k, inv_freq=inv)[0],
                       inkling_qk_norm_rope(tr.contiguous(), k, inv_freq=inv)[0])
    one = q[:1].expand(T, H, 128)
    assert torch.equal(inkling_qk_norm_rope(one, k, inv_freq=inv)[0],
                       inkling_qk_norm_rope(one.contiguous(), k, inv_freq=inv)[0])


def test_backward_is_the_same_every_time_and_matches_autograd(both_paths):
    T, H, K = 3000, 8, 2
    q, k, gq, gk = (_randn(T, n, 128, seed=i).cuda() for i, n in enumerate((H, K, H, K)))
    wq, wk = _dev(*_weights(torch.float32))
    inv = _inv_freq(128).cuda()
    a = inkling_qk_norm_rope_backward(gq, gk, q, k, wq, wk, inv_freq=inv)
    b = inkling_qk_norm_rope_backward(gq, gk, q, k, wq, wk, inv_freq=inv)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    out = inkling_qk_norm_rope(*leaves, inv_freq=inv)
    got = torch.autograd.grad(out, leaves, (gq, gk))
    assert all(torch.equal(x, y) for x, y in zip(a, got))
    # one weight shared by q and k gets the sum of both gradients; no gradient of k is asked for
    w = wq.clone().requires_grad_()
    qo, ko = inkling_qk_norm_rope(q, k, w, w, inv_freq=inv)
    (dw,) = torch.autograd.grad((qo, ko), (w,), (gq, gk))
    want = inkling_qk_norm_rope_backward(gq, gk, q, k, wq, wq, inv_freq=inv)
    assert torch.equal(dw, want[2] + want[3])


def test_empty_and_no_weight_gradients():
    e = torch.empty(0, 4, 128, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(128, device="cuda")
    qo, ko = inkling_qk_norm_rope(e, e, w, w)
    assert qo.shape == e.shape and ko.shape == e.shape
    dq, dk, dwq, dwk = inkling_qk_norm_rope_backward(e, e, e, e, w, w)
    assert dq.shape == e.shape and bool((dwq == 0).all()) and bool((dwk == 0).all())


def test_eps_of_any_kind(both_paths):
    """A whole number is an eps like any other; what is none is refused, rotation or not."""
    x = _randn(5, 2, 128, seed=7).cuda()
    inv = _inv_freq(64).cuda()
    for eps in (0, 1):
        got = inkling_qk_norm_rope(x, x, eps=eps, inv_freq=inv)[0]
        assert torch.equal(got, inkling_qk_norm_rope(x, x, eps=float(eps), inv_freq=inv)[0])
        want = oracle.norm_rope(_np(x), None, np.arange(5), eps, _np(inv), False)
        _check_rows(got, want, _np(inv), False)
    for eps in (-1.0, -1, -1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            inkling_qk_norm_rope(x, x, eps=eps, inv_freq=inv)
        with pytest.raises(ValueError, match="eps"):
            inkling_qk_norm_rope_backward(x, x, x, x, eps=eps, inv_freq=inv)


def test_refusals():
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    inv = torch.ones(64, dtype=torch.float64, device="cuda")
    w = torch.ones(128, device="cuda")
    for exc, msg, args, kw in (
            (TypeError, "bfloat16", (x.float(), x), {}),
            (ValueError, r"\[tokens, heads, 128\]", (x[:, :, :64], x), {}),
            (ValueError, "tokens and device", (x, x[:2]), {}),
            (ValueError, "neither", (x, x), dict(eps=None)),
            (ValueError, "without the norm", (x, x, w), dict(eps=None, inv_freq=inv)),
            (ValueError, "eps", (x, x), dict(eps=-1e-6)),
            (ValueError, "inv_freq", (x, x), dict(inv_freq=inv[:10])),
            (ValueError, "inv_freq", (x, x), dict(inv_freq=inv.cpu())),
            (TypeError, "inv_freq", (x, x), dict(inv_freq=inv.half())),
            (ValueError, "q_weight", (x, x, w[:64]), {}),
            (TypeError, "q_weight", (x, x, w.half()), {}),
            (TypeError, "differ in dtype", (x, x, w, w.bfloat16()), {}),
            (ValueError, "cu_seqlens_k needs", (x, x, None, None, None, cu), {}),
            (ValueError, "differ in length", (x, x, None, None, cu, torch.cat((cu, cu))), {}),
            (ValueError, "int32", (x, x, None, None, cu.long()), {})):
        with pytest.raises(exc, match=msg):
            inkling_qk_norm_rope(*args, **kw)
    with pytest.raises(ValueError, match="heads"):
        inkling_qk_norm_rope_backward(x[:, :1], x, x, x)


# --- append to the paged cache -------------------------------------------------------------------

def _paged_setup(lens_k, page_size, kv, seed, spare=3, strided=False):
    n_per = [-(-n // page_size) for n in lens_k]
    pages = sum(n_per) + spare
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens_k), max(n_per + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(n_per):
        table[b, :n] = perm[at:at + n]
        at += n
    shape = (pages, 2, page_size, kv, 128) if strided else (2, pages, page_size, kv, 128)
    both = _randn(*shape, seed=seed + 1)
    both.view(-1)[::7] = float("nan")  # whatever unused slots hold has to stay
    return table, both


def _same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


@pytest.mark.parametrize("lens_q,lens_k,page,heads,kv,rot,inter,wt,eps,strided", [
    ([1], [1], 16, 32, 8, 128, False, torch.bfloat16, 1e-6, False),
    ([1] * 5, [17, 16, 1, 33, 4096], 16, 8, 2, 64, True, torch.bfloat16, 1e-6, True),
    ([70, 0, 3, 128], [70, 9, 300, 129], 64, 4, 4, 128, False, torch.float32, 1e-6, False),
    ([5, 300], [5, 1000], 256, 0, 1, 32, False, None, 1e-6, True),
    ([3, 2], [100, 2], 32, 3, 3, 0, False, None, None, False),
])
def test_append(lens_q, lens_k, page, heads, kv, rot, inter, wt, eps, strided, both_paths):
    T = sum(lens_q)
    cu_q, cu_k = cu_from_lens(lens_q), cu_from_lens(lens_k)
    q, k, v = (_randn(T, n, 128, seed=i + 1) for i, n in enumerate((max(heads, 1), kv, kv)))
    wq, wk = _weights(wt)
    inv = _inv_freq(rot)
    table, both = _paged_setup(lens_k, page, kv, seed=11, strided=strided)
    dev = both.cuda()
    kc, vc = (dev[:, 0], dev[:, 1]) if strided else (dev[0], dev[1])
    dq, dk, dv, dwq, dwk, dtab, dcq, dck = _dev(q, k, v, wq, wk, table, cu_q, cu_k)
    kw = dict(k_weight=dwk, eps=eps, inv_freq=None if inv is None else inv.cuda(),
              interleaved=inter)
    if heads:
        kw.update(q=dq, q_weight=dwq)
    qo = inkling_kv_append(dk, dv, kc, vc, dtab, dcq, dck, **kw)
    pos = oracle.token_positions(T, cu_q.numpy(), cu_k.numpy())
    want_k = oracle.norm_rope(_np(k), _np(wk), pos, eps, _np(inv), inter)
    # the rows that belong somewhere, and nothing else
    mark = np.zeros(tuple(kc.shape[:2]))
    marked, _ = oracle.kv_append(mark, mark, np.ones(T), np.ones(T), table.numpy(), cu_q.numpy(),
                                 cu_k.numpy())
    assert marked.sum() == sum(lens_q)
    old_k, old_v = ((both[:, 0], both[:, 1]) if strided else (both[0], both[1]))
    untouched = torch.from_numpy(marked == 0)
    assert _same_bits(kc.cpu()[untouched], old_k[untouched])
    assert _same_bits(vc.cpu()[untouched], old_v[untouched])
    got_k, got_v = torch.zeros(T, kv, 128, dtype=torch.bfloat16), torch.zeros(T, kv, 128,
                                                                             dtype=torch.bfloat16)
    cu = cu_q.tolist()
    for b in range(len(lens_q)):
        for t in range(cu[b], cu[b + 1]):
            p = int(pos[t])
            got_k[t] = kc[int(table[b, p // page]), p % page].cpu()
            got_v[t] = vc[int(table[b, p // page]), p % page].cpu()
    assert _same_bits(got_v, v)
    _check_rows(got_k, want_k, _np(inv), inter, "keys")
    if heads:
        want_q = oracle.norm_rope(_np(q), _np(wq), pos, eps, _np(inv), inter)
        _check_rows(qo, want_q, _np(inv), inter, "queries")
    else:
        assert qo is None
    # the same step as the call without a cache, bit for bit
    if heads and (eps is not None or inv is not None):
        ref = inkling_qk_norm_rope(dq, dk, dwq, dwk, dcq, dck, eps=eps, inv_freq=kw["inv_freq"],
                                   interleaved=inter)
        assert torch.equal(ref[0], qo) and _same_bits(ref[1].cpu(), got_k)


def test_tokens_without_a_place_write_nothing(both_paths):
    """Table entries of -1 and past the cache, positions below 0 and past the table, and rows
    behind the last sequence."""
    page, kv = 16, 2
    lens_q, lens_k = [20, 4, 2, 3], [20, 2, 100, 3]
    T = sum(lens_q) + 5
    cu_q, cu_k = _dev(cu_from_lens(lens_q), cu_from_lens(lens_k))
    k, v, q = (_randn(T, n, 128, seed=i).cuda() for i, n in enumerate((kv, kv, 4)))
    table = torch.tensor([[0, -1, 7], [1, 1, 1], [2, 3, 4], [50, 2, 2]], dtype=torch.int32)
    cache = torch.full((2, 6, page, kv, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    q_out = torch.full_like(q, 3.0)
    inkling_kv_append(k, v, cache[0], cache[1], table.cuda(), cu_q, cu_k, q=q, q_out=q_out,
                      eps=None)
    # sequence 0: tokens 0..15 in page 0, 16..19 nowhere; sequence 1: positions -2, -1 nowhere,
    # 0 and 1 in page 1; sequence 2: positions 98, 99 past the table; sequence 3: page 50
    want = torch.full((6, page, kv, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    want[0], want[1, :2] = k[:16], k[22:24]
    assert torch.equal(cache[0], want)
    want[0], want[1, :2] = v[:16], v[22:24]
    assert torch.equal(cache[1], want)
    assert torch.equal(q_out[:29], q[:29]) and bool((q_out[29:] == 3.0).all())


def test_append_queries_in_place():
    T, H, K, page = 33, 4, 2, 16
    merged = _randn(T, (H + 2 * K) * 128, seed=2).cuda()
    q, k, v = (merged[:, a * 128:b * 128].view(T, b - a, 128)
               for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    table, both = _paged_setup([T], page, K, seed=4)
    kc, vc = both.cuda()
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    inv = _inv_freq(128).cuda()
    keep = merged.clone()
    want = inkling_kv_append(k, v, kc, vc, table.cuda(), cu, cu, q=q, inv_freq=inv)
    got = inkling_kv_append(k, v, kc, vc, table.cuda(), cu, cu, q=q, q_out=q, inv_freq=inv)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    assert torch.equal(merged[:, H * 128:], keep[:, H * 128:])


def test_append_refusals():
    T, H, K, page = 4, 2, 2, 16
    base = _randn(T, H + 2 * K, 128, seed=2).cuda()
    q, k, v = base[:, :H], base[:, H:H + K], base[:, H + K:]
    cache = torch.zeros(2, 3, page, K, 128, dtype=torch.bfloat16, device="cuda")
    kc, vc = cache
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")

    def call(k=k, v=v, kc=kc, vc=vc, table=table, cu_q=cu, cu_k=cu, **kw):
        return inkling_kv_append(k, v, kc, vc, table, cu_q, cu_k, **kw)

    for exc, msg, kw in (
            (ValueError, "needs cu_seqlens", dict(cu_k=None)),
            (ValueError, "heads", dict(v=v[:, :1])),
            (TypeError, "bfloat16", dict(kc=kc.float())),
            (ValueError, "num_pages, page_size", dict(kc=kc[:, :, :1])),
            (ValueError, "differ in shape", dict(vc=vc[:2])),
            (ValueError, "same memory", dict(vc=kc)),
            (ValueError, "page_size", dict(kc=kc[:, :8], vc=vc[:, :8])),
            (ValueError, "strides", dict(kc=kc.transpose(2, 3).contiguous().transpose(2, 3))),
            (ValueError, "block_table", dict(table=table.long())),
            (ValueError, "block_table", dict(table=torch.cat((table, table)))),
            (ValueError, "without q", dict(q_weight=torch.ones(128, device="cuda"))),
            (ValueError, "share no storage", dict(q=q, q_out=k)),
            (ValueError, "unit last stride", dict(q=q, q_out=torch.empty(
                T, 128, H, dtype=torch.bfloat16, device="cuda").transpose(1, 2)))):
        with pytest.raises(exc, match=msg):
            call(**kw)
