"""The operators in a row, as a layer calls them: serving (append with norm and rotation, then
decode behind the shared prefix with a bucketed bias; captured in a CUDA graph and replayed; on a
side stream) and training (norm and rotation, bucketed bias, attention, all gradients)."""
import numpy as np
import pytest
import torch

import oracle
from gpu_util import device_status_ok
from inkling_fa4 import (inkling_bucket_bias, inkling_bucket_bias_backward,
                         inkling_fa4_rel_attention, inkling_fa4_rel_attention_backward,
                         inkling_fa4_rel_attention_decode_shared_prefix,
                         inkling_fa4_rel_attention_triton, inkling_kv_append,
                         inkling_qk_norm_rope, inkling_qk_norm_rope_backward,
                         relative_bucket_starts)
from inkling_fa4.workloads import cu_from_lens

pytestmark = pytest.mark.gpu

H, K, R, PAGE = 8, 2, 128, 16


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert device_status_ok(), "a kernel abandoned a bounded wait"


def _randn(*shape, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(*shape, generator=g)).to(torch.bfloat16).cuda()


def _inv_freq():
    return (10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)).cuda()


class Server:
    """A prefix of 200 tokens prefilled once into shared pages, and B sequences behind it."""

    def __init__(self, B=5, prefix=208, room=64):
        self.B, self.prefix = B, prefix
        shared = prefix // PAGE
        own = room // PAGE
        pages = shared + B * own
        perm = torch.randperm(pages, generator=torch.Generator().manual_seed(0)).int().cuda()
        self.table = torch.empty(B, shared + own, dtype=torch.int32, device="cuda")
        self.table[:, :shared] = perm[:shared]
        self.table[:, shared:] = perm[shared:].view(B, own)
        self.cache = torch.full((2, pages, PAGE, K, 128), float("nan"), dtype=torch.bfloat16,
                                device="cuda")
        self.wq, self.wk = (1 + _randn(128, seed=i, std=0.2) for i in (1, 2))
        self.inv = _inv_freq()
        self.starts = torch.tensor(relative_bucket_starts(32, 128), dtype=torch.int32,
                                   device="cuda")
        self.bias_table = _randn(32, H, seed=3, std=0.5)
        self.step_kw = dict(k_weight=self.wk, inv_freq=self.inv)
        k, v = _randn(prefix, K, 128, seed=4), _randn(prefix, K, 128, seed=5)
        one = torch.tensor([0, prefix], dtype=torch.int32, device="cuda")
        inkling_kv_append(k, v, *self.cache, self.table[:1], one, one, **self.step_kw)
        self.cu_q = cu_from_lens([1] * B).cuda()
        self.cu_k = torch.empty(B + 1, dtype=torch.int32, device="cuda")
        self.qkv = torch.empty(B, (H + 2 * K) * 128, dtype=torch.bfloat16, device="cuda")

    def inputs(self, t, lens):
        self.qkv.copy_(_randn(self.B, (H + 2 * K) * 128, seed=100 + t))
        self.cu_k.copy_(cu_from_lens(lens))

    def step(self):
        q, k, v = (self.qkv[:, a * 128:b * 128].view(self.B, b - a, 128)
                   for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
        q = inkling_kv_append(k, v, *self.cache, self.table, self.cu_q, self.cu_k, q=q,
                              q_weight=self.wq, **self.step_kw)
        rel = inkling_bucket_bias(self.bias_table, self.starts, self.B, R)
        return q, inkling_fa4_rel_attention_decode_shared_prefix(
            q, *self.cache, rel, self.cu_q, self.cu_k, 1, self.prefix + 64, R, self.prefix,
            softmax_scale=0.1, block_table=self.table), rel

    def check(self, q, out, rel, lens):
        want, _, size = oracle.decode_paged(
            *(t.double().cpu().numpy() for t in (q, self.cache[0], self.cache[1], rel)), lens,
            self.table.cpu().numpy(), 0.1, R)
        tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -11) * size
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


def test_serving_steps():
    s = Server()
    for t in range(3):
        lens = [s.prefix + 1 + t + 7 * b for b in range(s.B)]
        if t == 0:  # the keys behind the prefix that earlier steps would have left
            for b in range(s.B):
                n = 7 * b
                if n:
                    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
                    ck = torch.tensor([0, s.prefix + n], dtype=torch.int32, device="cuda")
                    inkling_kv_append(_randn(n, K, 128, seed=50 + b), _randn(n, K, 128, seed=70 + b),
                                      *s.cache, s.table[b:b + 1], cu, ck, **s.step_kw)
        s.inputs(t, lens)
        q, out, rel = s.step()
        s.check(q, out, rel, lens)


def test_serving_step_in_a_graph_and_on_a_side_stream():
    s = Server()
    # whatever the captured call saw, a replay goes by what the buffers hold then
    s.cache[:, s.table[:, s.prefix // PAGE:].flatten().long()] = 0.25
    s.inputs(0, [s.prefix + 1] * s.B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            s.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = s.step()
    for t in (1, 2):
        lens = [s.prefix + 1 + (5 * b + t) % 60 for b in range(s.B)]
        s.inputs(t, lens)
        graph.replay()
        torch.cuda.synchronize()
        s.check(*captured, lens)
        got = [x.clone() for x in captured]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = s.step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def _training_inputs():
    lens = [100, 1, 60]
    T = sum(lens) + 3  # rows behind the last sequence
    cu = cu_from_lens(lens).cuda()
    merged = _randn(T, (H + 2 * K) * 128, seed=1)
    wq, wk = (1 + _randn(128, seed=i, std=0.2).float() for i in (2, 3))
    table = _randn(32, H, seed=4, std=0.5).float()
    starts = torch.tensor(relative_bucket_starts(32, 64), dtype=torch.int32, device="cuda")
    return lens, T, cu, merged, wq, wk, table, starts


def test_training_step():
    """Gradients of merged projection output, norm weights and bias table through autograd equal
    the explicit calls; the rows behind the last sequence have none."""
    lens, T, cu, merged, wq, wk, table, starts = _training_inputs()
    inv = _inv_freq()
    leaves = [t.clone().requires_grad_() for t in (merged, wq, wk, table)]
    m, lwq, lwk, lt = leaves
    # elementwise selection keeps the gradient of the rows behind the last sequence out of v's path
    q, k, v = (m[:, a * 128:b * 128].view(T, b - a, 128)
               for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    qn, kn = inkling_qk_norm_rope(q, k, lwq, lwk, cu, inv_freq=inv)
    rel = inkling_bucket_bias(lt, starts, T, 64, cu)
    args = (cu, cu, max(lens), max(lens), 64)
    n = sum(lens)
    out = inkling_fa4_rel_attention(qn[:n], kn[:n], v[:n], rel[:n], *args)
    dout = _randn(n, H, 128, seed=9)
    grads = torch.autograd.grad(out, leaves, dout)
    # explicit
    with torch.no_grad():
        qn, kn = inkling_qk_norm_rope(q, k, wq, wk, cu, inv_freq=inv)
        rel = inkling_bucket_bias(table, starts, n, 64)
        o, lse = inkling_fa4_rel_attention_triton(qn[:n], kn[:n], v[:n], rel, *args,
                                                  return_lse=True)
        dqn, dkn, dv, drel = inkling_fa4_rel_attention_backward(dout, qn[:n], kn[:n], v[:n], rel, o,
                                                                lse, *args)
        dq, dk, dwq, dwk = inkling_qk_norm_rope_backward(dqn, dkn, q[:n], k[:n], wq, wk, cu,
                                                         inv_freq=inv)
        dt = inkling_bucket_bias_backward(drel, starts, 32)
    assert torch.equal(out, o)
    assert torch.equal(grads[1], dwq) and torch.equal(grads[2], dwk)
    assert torch.equal(grads[0][:n], torch.cat([t.flatten(1) for t in (dq, dk, dv)], dim=1))
    assert bool((grads[0][n:] == 0).all())
    torch.testing.assert_close(grads[3], dt, rtol=1e-5, atol=1e-5)  # other chunks of tokens


def test_training_step_against_the_formulas():
    """The whole step against torch autograd in 64 bits on the CPU.  Intermediate tensors are
    rounded to bf16 between the operators (q, k, P, the output, their gradients), so the gradients
    agree to a few of those roundings: 2.5 % of the largest entry, as the attention's own gradient
    tests allow."""
    lens, T, cu, merged, wq, wk, table, starts = _training_inputs()
    n = sum(lens)
    inv = _inv_freq()
    leaves = [t.detach().double().cpu().requires_grad_() for t in (merged[:n], wq, wk, table)]
    m, dwq, dwk, dt = leaves
    pos = torch.cat([torch.arange(x) for x in lens]).double()
    angle = pos[:, None, None] * inv.cpu()

    def norm_rope(x, w):
        y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        a, b = y[..., :64], y[..., 64:]
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

    q = norm_rope(m[:, :H * 128].reshape(n, H, 128), dwq)
    k = norm_rope(m[:, H * 128:(H + K) * 128].reshape(n, K, 128), dwk)
    v = m[:, (H + K) * 128:].reshape(n, K, 128)
    bucket = torch.from_numpy(oracle.bucket_of(starts.cpu().numpy(), 64))
    outs, at = [], 0
    for s in lens:
        d = torch.arange(s)[:, None] - torch.arange(s)[None, :]
        bias = dt[bucket[d.clamp(0, 63)]].permute(2, 0, 1)
        bias = torch.where((d >= 0) & (d < 64), bias, torch.zeros_like(bias))
        kk, vv = (x[at:at + s].repeat_interleave(H // K, dim=1) for x in (k, v))
        x = torch.einsum("qhd,khd->hqk", q[at:at + s], kk) / 128 + bias
        p = x.masked_fill(d < 0, -float("inf")).softmax(-1)
        outs.append(torch.einsum("hqk,khd->qhd", p, vv))
        at += s
    dout = _randn(n, H, 128, seed=9)
    want = torch.autograd.grad(torch.cat(outs), leaves, dout.double().cpu())
    gl = [t.detach().clone().requires_grad_() for t in (merged, wq, wk, table)]
    gm = gl[0]
    gq, gk, gv = (gm[:n, a * 128:b * 128].view(n, b - a, 128)
                  for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    qn, kn = inkling_qk_norm_rope(gq, gk, gl[1], gl[2], cu, inv_freq=inv)
    rel = inkling_bucket_bias(gl[3], starts, n, 64, cu)
    out = inkling_fa4_rel_attention(qn, kn, gv, rel, cu, cu, max(lens), max(lens), 64)
    got = torch.autograd.grad(out, gl, dout)
    for g, w in zip((got[0][:n],) + got[1:], want):
        err = float((g.double().cpu() - w).abs().max())
        assert err <= 2.5e-2 * float(w.abs().max()), err


def test_training_gradients_in_a_graph():
    """The explicit gradient calls captured and replayed with new values, bit for bit; two graphs
    that were captured side by side do not disturb each other."""
    lens, T, cu, merged, wq, wk, table, starts = _training_inputs()
    inv = _inv_freq()
    q, k = merged[:, :H * 128].view(T, H, 128), merged[:, H * 128:(H + K) * 128].view(T, K, 128)
    drel = _randn(T, H, 64, seed=20)

    def step():
        g = inkling_qk_norm_rope_backward(q, k, q, k, wq, wk, cu, inv_freq=inv)
        return list(g) + [inkling_bucket_bias_backward(drel, starts, 32, cu_seqlens_q=cu)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    merged.copy_(_randn(*merged.shape, seed=21))
    drel.copy_(_randn(*drel.shape, seed=22))
    want = step()
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
