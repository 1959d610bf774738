"""Sequence offsets that are a column of a wider int32 tensor (stride 2): every attention entry point
reads the column, not the memory behind its first element.  The other column holds valid offsets too,
so a call that read them would give another result, not a fault."""
import pytest
import torch

from gpu_util import device_status_ok
from inkling_fa4 import (_ops, inkling_fa4_rel_attention_backward,
                         inkling_fa4_rel_attention_decode_shared_prefix,
                         inkling_fa4_rel_attention_decode_triton, inkling_fa4_rel_attention_triton)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert device_status_ok(), "a kernel abandoned a bounded wait"


def _randn(*shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _columns(values, others):
    """``values`` contiguous, and as column 0 of a tensor whose column 1 is ``others``."""
    flat = torch.tensor(values, dtype=torch.int32, device="cuda")
    both = torch.stack((flat, torch.tensor(others, dtype=torch.int32, device="cuda")), 1)
    assert both[:, 0].stride() == (2,)
    return flat, both[:, 0]


@pytest.mark.parametrize("path", [True, False], ids=["ops", "ctypes"])
@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_decode_and_shared_prefix(path, which):
    # read as contiguous: rows 0, 0, 1, 1 and key counts 80, 0, 90, 0
    cu_q, cu_q2 = _columns([0, 1, 2, 3, 4], [0, 1, 2, 3, 3])
    cu_k, cu_k2 = _columns([0, 80, 170, 270, 380], [80, 80 + 90, 270, 380, 380])
    kc, vc = (_randn(40, 16, 2, 128, seed=s) for s in (1, 2))
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(4, 10).contiguous()
    table[1:, :4] = table[0, :4].clone()
    q, rel = _randn(4, 8, 128, seed=3), _randn(4, 8, 64, seed=4)

    def calls(cu_q, cu_k):
        yield inkling_fa4_rel_attention_decode_shared_prefix(
            q, kc, vc, rel, cu_q, cu_k, 1, 110, 64, 64, block_table=table)
        yield inkling_fa4_rel_attention_decode_triton(
            q, kc, vc, rel, cu_q, cu_k, 1, 110, 64, block_table=table)

    before = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = path
    try:
        want = list(calls(cu_q, cu_k))
        got = list(calls(cu_q2 if which != "k" else cu_q, cu_k2 if which != "q" else cu_k))
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    finally:
        _ops.USE_TORCH_OPS = before


@pytest.mark.parametrize("path", [True, False], ids=["ops", "ctypes"])
def test_prefill_and_backward(path):
    # read as contiguous: sequences of 30 and 0 tokens, then 40
    cu, cu2 = _columns([0, 30, 70], [30, 70, 70])
    q, k, v = _randn(70, 4, 128, seed=1), _randn(70, 2, 128, seed=2), _randn(70, 2, 128, seed=3)
    rel, dout = _randn(70, 4, 32, seed=4), _randn(70, 4, 128, seed=5)
    before = _ops.USE_TORCH_OPS
    _ops.USE_TORCH_OPS = path
    try:
        want, got = [], []
        for outs, c in ((want, cu), (got, cu2)):
            out, lse = inkling_fa4_rel_attention_triton(q, k, v, rel, c, c, 40, 40, 32,
                                                        return_lse=True)
            outs += [out, lse]
            outs += inkling_fa4_rel_attention_backward(dout, q, k, v, rel, want[0], want[1], c, c,
                                                       40, 40, 32)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    finally:
        _ops.USE_TORCH_OPS = before
