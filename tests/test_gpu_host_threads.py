"""Calls from host threads that have made no CUDA call of their own yet (torch's autograd workers are
such threads): the tensor maps are encoded with the device's context bound."""
import threading

import pytest
import torch

from gpu_util import device_status_ok
from inkling_fa4 import inkling_fa4_rel_attention_decode_triton, inkling_fa4_rel_attention_triton
from inkling_fa4.workloads import make_case

pytestmark = pytest.mark.gpu


def test_first_cuda_call_of_a_thread():
    c = make_case([40, 9], [40, 9], 4, 2, 32, seed=1, device="cuda")
    d = make_case([1, 1], [64, 5], 4, 2, 32, seed=2, device="cuda")

    def prefill(out):
        inkling_fa4_rel_attention_triton(c.q, c.k, c.v, c.rel, c.cu_q, c.cu_k, 40, 40, 32, out=out)

    def decode(out):
        inkling_fa4_rel_attention_decode_triton(d.q, d.k, d.v, d.rel, d.cu_q, d.cu_k, 1, 64, 32,
                                                causal_align="bottom_right", out=out)

    for call, q in ((prefill, c.q), (decode, d.q)):
        want, got, errors = torch.empty_like(q), torch.zeros_like(q), []
        call(want)
        torch.cuda.synchronize()

        def body():
            try:
                call(got)
            except Exception as e:  # noqa: BLE001 (reported below, in the test's own thread)
                errors.append(e)

        t = threading.Thread(target=body)
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert not errors, errors
        assert torch.equal(got, want)
    assert device_status_ok()
