"""The wait of an eviction's blocks on one another is bounded: on a flag that nothing sets it runs out after
its limit, sets its bit of the status word and no other, and leaves the context usable."""
import pytest
import torch

from inkling_fa4 import _lib
from long_context_cases import Case
from test_gpu_kv_evict import _check_evict, _mass

pytestmark = pytest.mark.gpu


def test_wait_runs_out_and_reports():
    L = _lib.lib()
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.read_device_status(stream, clear=True) == 0
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    _lib.check(L.ifa4_selftest_evict_wait(20_000_000, stream))  # 20 ms limit
    e1.record()
    assert _lib.read_device_status(stream, clear=True) == 128  # synchronises
    assert 15.0 <= e0.elapsed_time(e1) < 150.0
    c = Case([1, 1], [300, 170], 8, 2, 16, 8, seed=91)
    _check_evict(c, _mass(c), 70, 3, 20)
    assert _lib.read_device_status(stream, clear=True) == 0


@pytest.mark.parametrize("bad", [0, -5, 2_000_000_000])
def test_bad_limits_are_refused(bad):
    assert _lib.lib().ifa4_selftest_evict_wait(bad, None) == _lib.IFA4_ERR_INVALID_ARGUMENT
