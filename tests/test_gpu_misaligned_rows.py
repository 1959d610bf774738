"""Inputs that are contiguous but start between two 16-byte boundaries (a slice of a flat buffer) are
copied like every other layout the kernels do not read in place."""
import pytest
import torch

from inkling_fa4 import (_ops, inkling_fa4_rel_attention_backward,
                         inkling_fa4_rel_attention_decode_shared_prefix,
                         inkling_fa4_rel_attention_decode_triton, inkling_fa4_rel_attention_triton,
                         inkling_kv_append, inkling_qk_norm_rope, inkling_qk_norm_rope_backward,
                         inkling_rel_logits)

pytestmark = pytest.mark.gpu


def _pair(*shape):
    """A tensor, and the same values 2 bytes behind a 16-byte boundary."""
    t = torch.randn(*shape, device="cuda").to(torch.bfloat16)
    pool = torch.empty(t.numel() + 8, dtype=torch.bfloat16, device="cuda")
    off = pool[1:1 + t.numel()].view(shape)
    off.copy_(t)
    assert off.is_contiguous() and off.data_ptr() % 16 == 2
    return t, off


@pytest.fixture(params=[True, False], ids=["ops", "ctypes"], autouse=True)
def path(request):
    before = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = request.param
    yield
    _ops.USE_TORCH_OPS = before


@pytest.mark.parametrize("T", [1, 40])
def test_attention(T):
    q, k, v, rel, dout = (_pair(T, h, d) for h, d in ((4, 128), (2, 128), (2, 128), (4, 16), (4, 128)))
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    outs = []
    for i in (0, 1):
        out, lse = inkling_fa4_rel_attention_triton(q[i], k[i], v[i], rel[i], cu, cu, T, T, 16,
                                                    return_lse=True)
        outs.append([out, lse, *inkling_fa4_rel_attention_backward(
            dout[i], q[i], k[i], v[i], rel[i], out, lse, cu, cu, T, T, 16)])
    for a, b in zip(*outs):  # the bias is read in another way: the same sums in another order at most
        torch.testing.assert_close(a, b, atol=1e-6, rtol=2 ** -7)


def test_decode():
    q, k, v, rel = _pair(1, 4, 128), _pair(50, 2, 128), _pair(50, 2, 128), _pair(1, 4, 16)
    one = torch.arange(2, dtype=torch.int32, device="cuda")
    a, b = (inkling_fa4_rel_attention_decode_triton(q[i], k[i], v[i], rel[i], one, 50 * one, 1, 50, 16)
            for i in (0, 1))
    assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 33])
def test_operators(T):
    q, k, v, gq, gk = (_pair(T, h, 128) for h in (4, 2, 2, 4, 2))
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    inv = (100.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).cuda()
    w = torch.ones(128, device="cuda")
    table = torch.arange(3, dtype=torch.int32, device="cuda").view(1, 3)
    outs = []
    for i in (0, 1):
        caches = [torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        got = inkling_kv_append(k[i], v[i], *caches, table, cu, cu, q=q[i], q_weight=w, k_weight=w,
                                inv_freq=inv)
        outs.append([got, *caches, *inkling_qk_norm_rope(q[i], k[i], w, w, inv_freq=inv),
                     *inkling_qk_norm_rope_backward(gq[i], gk[i], q[i], k[i], w, w, inv_freq=inv)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_rel_logits():
    r, w = _pair(20, 4, 16), _pair(16, 64)
    cu = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    assert torch.equal(inkling_rel_logits(r[0], w[0], cu), inkling_rel_logits(r[1], w[1], cu))


def test_shared_prefix():
    q = _pair(2, 4, 128)
    kc, vc = (torch.randn(4, 16, 2, 128, device="cuda").to(torch.bfloat16) for _ in range(2))
    rel = torch.randn(2, 4, 16, device="cuda").to(torch.bfloat16)
    cu = torch.arange(3, dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1, 2], [0, 1, 3]], dtype=torch.int32, device="cuda")
    a, b = (inkling_fa4_rel_attention_decode_shared_prefix(x, kc, vc, rel, cu, cu * 40, 1, 40, 16, 32,
                                                           block_table=table) for x in q)
    assert torch.equal(a, b)
    odd = _pair(4, 16, 2, 128)[1]  # a cache is never copied
    with pytest.raises(ValueError, match="16-byte alignment"):
        inkling_fa4_rel_attention_decode_shared_prefix(q[0], odd, vc, rel, cu, cu * 40, 1, 40, 16, 32,
                                                       block_table=table)
