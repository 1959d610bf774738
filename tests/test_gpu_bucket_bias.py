"""Bias by distance buckets on the GPU and its gradient against the 64-bit oracle.

The bias is a table value rounded once to bf16: equal to torch's rounding bit for bit.  The
gradient adds exact bf16 values in fp32; the longest chain of additions is under 512 at these sizes
(at most 32 tokens a lane, 16 lanes, 128 columns a lane of a bucket of up to 1024, 3 shuffles, 40
slots a thread, 32 threads), so it is off by at most 512 * 2^-24 of the sum of sizes, and 2^-8 of
itself more where it is rounded to bf16."""
import numpy as np
import pytest
import torch

import oracle
from gpu_util import device_status_ok
from inkling_fa4 import (_ops, inkling_bucket_bias, inkling_bucket_bias_backward,
                         inkling_fa4_rel_attention, inkling_fa4_rel_attention_triton,
                         relative_bucket_starts)
from inkling_fa4.workloads import cu_from_lens, make_case

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


def _table(buckets, heads, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(buckets, heads, generator=g).to(dtype)


def _check_grad(got, drel, starts, tokens=None):
    want, size = oracle.bucket_bias_grad(drel.double().cpu().numpy(), starts, tokens)
    tol = 512 * 2.0 ** -24 * size
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
    err = np.abs(got.double().cpu().numpy() - want) - tol
    assert err.max() <= 0, err.max()


CASES = [  # tokens, heads, rel_extent, starts
    (128, 4, 128, relative_bucket_starts(32, 128)),
    (1, 1, 1, [0]),
    (0, 3, 64, relative_bucket_starts(8, 64)),
    (1000, 5, 100, relative_bucket_starts(20, 500)),
    (777, 3, 129, relative_bucket_starts(32, 128)),
    (333, 32, 1024, relative_bucket_starts(64, 1024)),
    (50, 2, 2500, relative_bucket_starts(128, 1024)),
    (5000, 8, 200, list(range(200))),               # one bucket a distance
    (300, 2, 64, [3, 10, 10, 500]),                 # late first start, an empty bucket, one beyond
    (64, 40, 8, [0, 4]),
    (20, 1, 9000, [0, 8999]),
    (600, 32, 100, relative_bucket_starts(20, 100)),   # heads one behind the other, read across
    (513, 40, 129, relative_bucket_starts(32, 128)),
    (100, 9, 24, relative_bucket_starts(8, 24)),
    (70, 6, 20, relative_bucket_starts(8, 24)),
]


@pytest.mark.parametrize("T,H,R,starts", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bias_and_gradient(T, H, R, starts, dtype):
    table = _table(len(starts), H, 1, dtype)
    st = torch.tensor(starts, dtype=torch.int32)
    rel = inkling_bucket_bias(table.cuda(), st.cuda(), T, R)
    assert rel.shape == (T, H, R) and (T < 2 or rel.stride(0) == 0)
    if T:
        want = table[torch.from_numpy(oracle.bucket_of(starts, R))].t().to(torch.bfloat16)
        assert torch.equal(rel[T - 1].cpu(), want)
    g = torch.Generator().manual_seed(2)
    drel = (0.1 * torch.randn(T, H, R, generator=g)).to(torch.bfloat16)
    got = inkling_bucket_bias_backward(drel.cuda(), st.cuda(), len(starts), dtype=dtype)
    assert got.shape == table.shape and got.dtype == dtype
    _check_grad(got, drel, starts)


def test_gradient_layouts(both_paths):
    """Wider buffers, odd offsets, head and token orders, broadcast gradients, padded tokens."""
    starts = relative_bucket_starts(16, 100)
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(300, 6, 150, generator=g).to(torch.bfloat16).cuda()
    one = wide[:1].expand(300, 6, 150)
    for drel in (wide[:, :, :128], wide[:, :, 1:129], wide[:, :, 2:100], wide[:, ::2, :104],
                 wide.transpose(0, 1), wide.permute(0, 2, 1)[:, :128].permute(0, 2, 1),
                 wide.transpose(1, 2).contiguous().transpose(1, 2), one,
                 wide[:, :, :1].expand(300, 6, 128)):
        _check_grad(inkling_bucket_bias_backward(drel, st, 16), drel, starts)
    for lens in ([100, 57], [300], [0], [0, 0, 1], [1000]):
        cu = cu_from_lens(lens).cuda()
        bad = wide.clone()
        bad[min(sum(lens), 300):] = float("nan")
        _check_grad(inkling_bucket_bias_backward(bad, st, 16, cu_seqlens_q=cu), wide, starts,
                    min(sum(lens), 300))


def test_table_layouts_and_determinism(both_paths):
    starts = relative_bucket_starts(16, 100)
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    table = _table(16, 8, 4, torch.float32).cuda()
    want = inkling_bucket_bias(table, st, 4, 128)
    wide = torch.zeros(16, 20, device="cuda")
    wide[:, 3:11] = table
    assert torch.equal(inkling_bucket_bias(wide[:, 3:11], st, 4, 128), want)
    assert torch.equal(inkling_bucket_bias(table.t().contiguous().t(), st, 4, 128), want)
    g = torch.Generator().manual_seed(3)
    drel = torch.randn(20000, 8, 128, generator=g).to(torch.bfloat16).cuda()
    a, b = (inkling_bucket_bias_backward(drel, st, 16) for _ in range(2))
    assert torch.equal(a, b)


def test_infinite_gradients_stay_in_their_bucket():
    starts = [0, 10, 20]
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    drel = torch.zeros(40, 2, 64, dtype=torch.bfloat16, device="cuda")
    drel[7, 1, 12] = float("inf")
    drel[9, 0, 3] = float("nan")
    got = inkling_bucket_bias_backward(drel, st, 3).cpu()
    assert torch.isnan(got[0, 0]) and got[1, 1] == float("inf")
    assert got[0, 1] == 0 and bool((got[2] == 0).all()) and got[1, 0] == 0


def test_through_the_attention_and_its_gradient():
    """table -> bias -> attention -> gradient of the table, against the same through an explicit
    [tokens, heads, rel_extent] bias: the attention sees equal bits, and the table's gradient is
    that of its own d rel_logits."""
    lens = [150, 1, 77]
    c = make_case(lens, lens, 4, 2, 64, seed=5, device="cuda")
    starts = relative_bucket_starts(16, 64)
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    table = _table(16, 4, 6, torch.float32).cuda().requires_grad_()
    rel = inkling_bucket_bias(table, st, c.q.shape[0], 64, c.cu_q)
    args = (c.cu_q, c.cu_k, c.max_q, c.max_k, 64)
    out = inkling_fa4_rel_attention(c.q, c.k, c.v, rel, *args)
    full = rel.detach().contiguous().requires_grad_()
    ref = inkling_fa4_rel_attention_triton(c.q, c.k, c.v, full.detach(), *args)
    assert torch.equal(out, ref)
    dout = torch.randn_like(out)
    (dtable,) = torch.autograd.grad(out, (table,), dout)
    (drel,) = torch.autograd.grad(inkling_fa4_rel_attention(c.q, c.k, c.v, full, *args), (full,),
                                  dout)
    assert torch.equal(dtable, inkling_bucket_bias_backward(drel, st, 16, cu_seqlens_q=c.cu_q))
    _check_grad(dtable, drel, starts)


def test_refusals():
    st = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    table = torch.zeros(2, 3, device="cuda")
    drel = torch.zeros(5, 3, 16, dtype=torch.bfloat16, device="cuda")
    for exc, msg, call in (
            (TypeError, "bfloat16 or float32", lambda: inkling_bucket_bias(table.half(), st, 5, 16)),
            (ValueError, "starts", lambda: inkling_bucket_bias(table, st.long(), 5, 16)),
            (ValueError, "starts", lambda: inkling_bucket_bias(table, st.cpu(), 5, 16)),
            (ValueError, "buckets", lambda: inkling_bucket_bias(table[:1], st, 5, 16)),
            (ValueError, "rel_extent", lambda: inkling_bucket_bias(table, st, 5, 0)),
            (ValueError, "total_q", lambda: inkling_bucket_bias(table, st, -1, 16)),
            (ValueError, "1024", lambda: inkling_bucket_bias(table, torch.zeros(
                1025, dtype=torch.int32, device="cuda"), 5, 16)),
            (TypeError, "bfloat16", lambda: inkling_bucket_bias_backward(drel.float(), st, 2)),
            (ValueError, "2 starts", lambda: inkling_bucket_bias_backward(drel, st, 3)),
            (ValueError, "total_q, n_heads", lambda: inkling_bucket_bias_backward(drel[0], st, 2)),
            (TypeError, "table must be", lambda: inkling_bucket_bias_backward(
                drel, st, 2, dtype=torch.float16)),
            (ValueError, "cu_seqlens_q", lambda: inkling_bucket_bias_backward(
                drel, st, 2, cu_seqlens_q=st.long()))):
        with pytest.raises(exc, match=msg):
            call()
