"""The operators next to the attention where calls go wrong elsewhere: offsets beyond 32 bits, NaN
keys, several calls at once, the debug build, autograd with leaves that an eager graph holds."""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from gpu_util import device_status_ok
from inkling_fa4 import (_lib, inkling_bucket_bias, inkling_bucket_bias_backward,
                         inkling_fa4_rel_attention_decode_shared_prefix,
                         inkling_fa4_rel_attention_decode_triton, inkling_kv_append,
                         inkling_qk_norm_rope, inkling_qk_norm_rope_backward,
                         relative_bucket_starts)

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
DEBUG_LIB = os.path.join(os.path.dirname(_lib.LIB_PATH), "libinkling_fa4_debug.so")


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert device_status_ok(), "a kernel abandoned a bounded wait"


def _randn(*shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (std * torch.randn(*shape, generator=g, device="cuda")).to(torch.bfloat16)


def _cu(*lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")


def _inv(n=64):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).cuda()


def test_cache_beyond_32_bit_offsets():
    """A cache of more than 2^31 elements: tokens appended to its last pages are found there by the
    shared-prefix decode, and the result equals that of a small cache, bit for bit."""
    K, page, prefix = 2, 16, 96
    pages = (1 << 31) // (page * K * 128) + 64
    k, v, q = _randn(prefix + 4, K, 128, seed=1), _randn(prefix + 4, K, 128, seed=2), \
        _randn(2, 8, 128, seed=3)
    rel = _randn(2, 8, 128, seed=4)
    outs = []
    for n in (16, pages):
        cache = [torch.empty(n, page, K, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        last = torch.arange(n - 8, n, dtype=torch.int32, device="cuda").flip(0)
        table = torch.stack((last, last)).contiguous()
        table[1, 6] = last[7]
        inkling_kv_append(k[:prefix], v[:prefix], *cache, table[:1], _cu(prefix), _cu(prefix),
                          inv_freq=_inv())
        inkling_kv_append(k[prefix:], v[prefix:], *cache, table, _cu(3, 1),
                          _cu(prefix + 3, prefix + 1), inv_freq=_inv())
        outs.append(inkling_fa4_rel_attention_decode_shared_prefix(
            q, *cache, rel, _cu(1, 1), _cu(prefix + 3, prefix + 1), 1, prefix + 3, 128, prefix,
            softmax_scale=0.1, block_table=table))
        outs.append(inkling_fa4_rel_attention_decode_triton(
            q, *cache, rel, _cu(1, 1), _cu(prefix + 3, prefix + 1), 1, prefix + 3, 128,
            softmax_scale=0.1, causal_align="bottom_right", block_table=table))
        del cache
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    torch.testing.assert_close(outs[2].float(), outs[3].float(), atol=2e-2, rtol=2e-2)


def test_rows_beyond_32_bit_offsets():
    T, H = (1 << 31) // (4 * 128) + 1000, 4
    q = torch.empty(T, H, 128, dtype=torch.bfloat16, device="cuda")
    q[:1000], q[-1000:] = _randn(1000, H, 128, seed=5), _randn(1000, H, 128, seed=6)
    q[1000:-1000] = 1.0
    k = q[:, :1]
    qo, ko = inkling_qk_norm_rope(q, k, inv_freq=_inv())
    tail = slice(T - 1000, T)
    cu_q, cu_k = _cu(1000), _cu(T)
    want = inkling_qk_norm_rope(q[tail], k[tail], None, None, cu_q, cu_k, inv_freq=_inv())
    assert torch.equal(qo[tail], want[0]) and torch.equal(ko[tail], want[1])
    del ko
    dq, _, _, _ = inkling_qk_norm_rope_backward(qo, qo[:, :1], q, k, inv_freq=_inv())
    gwant = inkling_qk_norm_rope_backward(qo[tail], qo[tail, :1], q[tail], k[tail], None, None, cu_q,
                                          cu_k, inv_freq=_inv())
    assert torch.equal(dq[tail], gwant[0])


def test_gradient_of_more_than_2_31_logits():
    """Ones: every partial sum is a whole number below 2^24 until the last additions, whose result
    has at most 2^-24 of rounding each (fewer than 64 of them)."""
    T, H, R = 36000, 64, 1024
    starts = relative_bucket_starts(32, 1024)
    drel = torch.ones(T, H, R, dtype=torch.bfloat16, device="cuda")
    got = inkling_bucket_bias_backward(drel, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                                       32)
    width = torch.tensor([b - a for a, b in zip(starts, starts[1:] + [R])], dtype=torch.float64)
    want = (width * T)[:, None].expand(32, H)
    assert bool(((got.double().cpu() - want).abs() <= 64 * 2.0 ** -24 * want).all())


def test_nan_in_a_prefix_key_reaches_only_the_rows_that_see_it():
    prefix, page = 128, 16
    kc, vc = (_randn(20, page, 2, 128, seed=s) for s in (7, 8))
    kc[2, 3, 1, 5] = float("nan")  # KV head 1, key 35
    table = torch.arange(10, dtype=torch.int32, device="cuda").expand(3, 10).contiguous()
    q, rel = _randn(3, 8, 128, seed=9), _randn(3, 8, 64, seed=10)
    out = inkling_fa4_rel_attention_decode_shared_prefix(
        q, kc, vc, rel, _cu(1, 1, 1), _cu(130, 140, 160), 1, 160, 64, prefix, block_table=table)
    assert bool(torch.isfinite(out[:, :4].float()).all())
    assert bool(torch.isnan(out[:, 4:].float()).all())


def test_calls_at_the_same_time():
    """Two batches on two streams, each with its own workspace, interleaved many times."""
    kc, vc = (_randn(600, 16, 2, 128, seed=s) for s in (1, 2))
    g = torch.Generator().manual_seed(3)
    jobs = []
    for n, prefix in ((5, 1024), (70, 2048)):
        table = torch.randperm(600, generator=g)[:160].int().cuda().expand(n, 160).contiguous()
        lens = [prefix + 1 + (37 * b) % 400 for b in range(n)]
        args = (_randn(n, 8, 128, seed=n), kc, vc, _randn(n, 8, 128, seed=n + 1), _cu(*[1] * n),
                _cu(*lens), 1, max(lens), 128, prefix)
        jobs.append((args, dict(block_table=table, softmax_scale=0.1)))
    want = [inkling_fa4_rel_attention_decode_shared_prefix(*a, **kw) for a, kw in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(20):
        for i, (a, kw) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                got[i].append(inkling_fa4_rel_attention_decode_shared_prefix(*a, **kw))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, x) for x in outs)


def test_gradients_in_a_graph_beside_an_eager_graph_of_the_same_leaves():
    """The explicit gradient calls can be captured while an eager autograd graph of the same tensors
    is alive (they make no autograd nodes), and that graph still runs afterwards."""
    q, k = _randn(40, 4, 128, seed=1).requires_grad_(), _randn(40, 2, 128, seed=2).requires_grad_()
    w = torch.ones(128, device="cuda", requires_grad=True)
    table = torch.zeros(8, 4, device="cuda", requires_grad=True)
    starts = torch.arange(8, dtype=torch.int32, device="cuda")
    alive = inkling_qk_norm_rope(q, k, w, w, inv_freq=_inv())
    bias = inkling_bucket_bias(table, starts, 40, 16)
    gq, gk, drel = _randn(40, 4, 128, seed=3), _randn(40, 2, 128, seed=4), _randn(40, 4, 16, seed=5)

    def explicit():
        return (*inkling_qk_norm_rope_backward(gq, gk, q, k, w, w, inv_freq=_inv_held),
                inkling_bucket_bias_backward(drel, starts, 8))

    _inv_held = _inv()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        explicit()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = explicit()
    graph.replay()
    dq, dk, dw, dt = torch.autograd.grad((*alive, bias), (q, k, w, table), (gq, gk, drel))
    torch.cuda.synchronize()
    assert torch.equal(captured[0], dq) and torch.equal(captured[1], dk)
    assert torch.equal(captured[2] + captured[3], dw) and torch.equal(captured[4], dt)


def test_plain_calls_hold_nothing_and_make_no_autograd_nodes():
    """The calls that skip the Python checks: outputs need no gradient whatever the inputs do, no
    reference or memory is left behind, and threads may call at the same time."""
    q, k = _randn(40, 4, 128, seed=1).requires_grad_(), _randn(40, 2, 128, seed=2)
    w = torch.nn.Parameter(torch.ones(128, device="cuda"))
    table, starts = _randn(8, 4, seed=3), torch.arange(8, dtype=torch.int32, device="cuda")
    inv = _inv()

    def calls():
        return (*_lib.plain_call("qk_norm_rope", q, k, w, w, inv, None, None, False, 1e-6),
                *_lib.plain_call("bucket_bias", table, starts, 40, 16))

    first = calls()
    assert not any(t.requires_grad or t.grad_fn is not None for t in first)
    assert first[2].shape == (40, 4, 16) and first[2].stride() == (0, 16, 1)
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(first, calls()))
    counts = [sys.getrefcount(t) for t in (q, k, w, inv, table, starts, None)]
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()

    def many(_):
        for _ in range(200):
            got = calls()
        return all(torch.equal(a, b) for a, b in zip(first, got))

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(many, range(4)))
    del pool
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == held
    assert [sys.getrefcount(t) for t in (q, k, w, inv, table, starts, None)] == counts


def run_debug_cases():
    """Every kernel of the operators on odd sizes; the outputs and the device status word."""
    out = {}
    q, k, v = (_randn(77, n, 128, seed=n) for n in (6, 3, 2))
    w = torch.ones(128, device="cuda") * 1.5
    cu_q, cu_k = _cu(30, 40), _cu(35, 90)
    for inter in (False, True):
        kw = dict(inv_freq=_inv(24), interleaved=inter)
        out[f"q{inter}"], out[f"k{inter}"] = inkling_qk_norm_rope(q, k, w, w, cu_q, cu_k, **kw)
        for i, t in enumerate(inkling_qk_norm_rope_backward(q, k, q, k, w, w, cu_q, cu_k, **kw)):
            out[f"g{i}{inter}"] = t
    cache = torch.zeros(2, 40, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    table = torch.arange(20, dtype=torch.int32, device="cuda").view(2, 10).contiguous()
    table[1, :4] = table[0, :4]
    out["append"] = inkling_kv_append(v[:70], v[:70], *cache, table, cu_q, cu_k, q=q[:70],
                                      inv_freq=_inv(8))
    out["cache"] = cache
    for heads, prefix in ((8, 33), (2, 64)):
        out[f"prefix{heads}"] = inkling_fa4_rel_attention_decode_shared_prefix(
            _randn(2, heads, 128, seed=1), *cache, _randn(2, heads, 50, seed=2), _cu(1, 1), cu_k, 1,
            90, 50, prefix, block_table=table)
    starts = torch.tensor(relative_bucket_starts(20, 90), dtype=torch.int32, device="cuda")
    out["bias"] = inkling_bucket_bias(_randn(20, 5, seed=3), starts, 1, 77)
    for r in (77, 128):
        out[f"dbias{r}"] = inkling_bucket_bias_backward(_randn(300, 5, r, seed=4), starts, 20)
    torch.cuda.synchronize()
    status = _lib.read_device_status(torch.cuda.current_stream().cuda_stream)
    return {n: t.detach().cpu() for n, t in out.items()}, status, _lib.LIB_PATH


@pytest.mark.skipif(not os.path.exists(DEBUG_LIB), reason="debug build not built")
def test_debug_build_reports_no_failed_check_and_matches_release(tmp_path):
    dst = str(tmp_path / "debug.pt")
    code = ("import sys; sys.path[:0] = [%r, %r, %r]; import torch, test_gpu_operators_edges as t; "
            "o = t.run_debug_cases(); torch.save({'outs': o[0], 'status': o[1], 'lib': o[2]}, %r)"
            % (HERE, os.path.dirname(HERE),
               os.path.join(os.path.dirname(HERE), "inkling-fa4-relative-attention_b200"), dst))
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, INKLING_FA4_LIB="debug"),
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    dbg = torch.load(dst)
    assert dbg["lib"].endswith("libinkling_fa4_debug.so") and dbg["status"] == 0
    outs, status, path = run_debug_cases()
    assert status == 0 and path.endswith("libinkling_fa4.so")
    for n, t in outs.items():
        torch.testing.assert_close(dbg["outs"][n], t, atol=0, rtol=0, msg=n)
