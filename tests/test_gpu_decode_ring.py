"""The decode kernel's ring of K/V stages: a stage may be refilled only when its last fragments have
been read.  The own keys of many sequences (up to 15 tiles each) beside a prefix kernel of many CTAs,
where a release that is not ordered behind the reads shows in most calls; the result depends neither on
the number of those CTAs (all but the first hold no keys and have weight 0) nor on the call."""
import pytest
import torch

from gpu_util import device_status_ok
from inkling_fa4 import (inkling_fa4_rel_attention_decode_shared_prefix,
                         inkling_fa4_rel_attention_decode_triton)

pytestmark = pytest.mark.gpu


def _batch(batch, prefix, page, most):
    g = torch.Generator(device="cuda").manual_seed(batch)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)

    own = [1 + 389 * b % most for b in range(batch)]
    lens = torch.tensor([prefix + n for n in own])
    shared, width = prefix // page, -(-int(lens.max()) // page)
    perm = torch.randperm(shared + batch * (width - shared), generator=g, device="cuda").int()
    table = torch.cat((perm[:shared].expand(batch, shared),
                       perm[shared:].view(batch, width - shared)), 1).contiguous()
    kc, vc = (randn(len(perm), page, 8, 128) for _ in range(2))
    cu_q = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    cu_k = torch.cat((torch.zeros(1, dtype=torch.int64), lens.cumsum(0))).int().cuda()
    args = (randn(batch, 32, 128), kc, vc, 0.5 * randn(batch, 32, 128), cu_q, cu_k, 1, int(lens.max()),
            128)
    return args, dict(softmax_scale=128 ** -0.5, block_table=table, return_lse=True)


@pytest.mark.parametrize("splits", [2, 16, 50])
def test_beside_a_prefix_kernel_of_many_ctas(splits):
    args, kw = _batch(109, 64, 64, 939)
    want = inkling_fa4_rel_attention_decode_shared_prefix(*args, 64, prefix_splits=1, num_splits=1,
                                                          **kw)
    for _ in range(30):
        got = inkling_fa4_rel_attention_decode_shared_prefix(*args, 64, prefix_splits=splits,
                                                             num_splits=1, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # the plain decode merges nothing: its rounding differs, its dims do not
    plain = inkling_fa4_rel_attention_decode_triton(*args, causal_align="bottom_right", num_splits=1,
                                                    **kw)
    torch.testing.assert_close(want[0].float(), plain[0].float(), atol=4e-3, rtol=2e-2)
    assert device_status_ok(), "a kernel abandoned a bounded wait"


def test_the_plain_decode_repeats_itself():
    args, kw = _batch(128, 0, 16, 2048)
    want = inkling_fa4_rel_attention_decode_triton(*args, causal_align="bottom_right", **kw)
    for _ in range(30):
        got = inkling_fa4_rel_attention_decode_triton(*args, causal_align="bottom_right", **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
