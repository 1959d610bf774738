"""The long-context kernels in the index-checking debug build: no check fails, and the outputs are those
of the release build, bit for bit."""
import os
import subprocess
import sys

import pytest
import torch

from inkling_fa4 import (_lib, inkling_fa4_rel_attention_decode_pages, inkling_kv_attention_mass,
                         inkling_kv_evict, inkling_kv_page_bounds, inkling_kv_page_scores,
                         inkling_kv_select_pages)
from long_context_cases import Case

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
DEBUG_LIB = os.path.join(os.path.dirname(_lib.LIB_PATH), "libinkling_fa4_debug.so")


def run_cases():
    """Outputs, the status word and the library's path."""
    outs = {}
    cases = [("single", Case([1, 0, 1, 1], [700, 40, 33, 1], 8, 2, 16, 50, seed=1, padding=2), (-1, -1)),
             ("chunks", Case([40, 3, 150], [40, 300, 700], 32, 1, 64, 100, seed=2), (300, 0)),
             ("rows before the keys", Case([9, 2], [4, 90], 6, 6, 16, 20, seed=3), (-1, -1))]
    for name, c, window in cases:
        kw = dict(block_table=c.table)
        more = (c.cu_q, c.cu_k, c.max_q, c.max_k, c.rel_extent)
        bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
        scores = inkling_kv_page_scores(c.q, bounds, c.rel, c.cu_q, c.cu_k, c.max_q, c.rel_extent,
                                        c.page_size, window, first_pages=1, last_pages=1, **kw)
        pages = inkling_kv_select_pages(scores, 5)
        for splits in (1, 3, 9):
            out, lse = inkling_fa4_rel_attention_decode_pages(c.q, c.k, c.v, c.rel, *more, pages, window,
                                                              num_splits=splits, return_lse=True, **kw)
            outs[f"{name}: attention, {splits}"], outs[f"{name}: lse, {splits}"] = out, lse
        mass = inkling_kv_attention_mass(c.q, c.k, c.rel, lse, *more, window, **kw)
        outs[f"{name}: bounds"], outs[f"{name}: scores"], outs[f"{name}: pages"] = bounds, scores, pages
        outs[f"{name}: mass"] = mass
        kept, left, cu = inkling_kv_evict(c.k, c.v, mass, c.table, c.cu_k, 70, first=2, recent=9)
        outs.update({f"{name}: kept": kept, f"{name}: left": left, f"{name}: cu": cu,
                     f"{name}: k": c.k, f"{name}: v": c.v})
    outs = {k: v.cpu() for k, v in outs.items()}
    status = _lib.read_device_status(torch.cuda.current_stream().cuda_stream, clear=True)
    return outs, status, _lib.LIB_PATH


@pytest.mark.skipif(not os.path.exists(DEBUG_LIB), reason="debug build not built")
def test_debug_build_reports_no_failed_check_and_matches_release(tmp_path):
    dst = str(tmp_path / "debug.pt")
    path = os.pathsep.join([HERE, os.path.dirname(os.path.dirname(os.path.dirname(_lib.LIB_PATH)))])
    env = dict(os.environ, INKLING_FA4_LIB="debug", PYTHONPATH=path)
    r = subprocess.run([sys.executable, os.path.abspath(__file__), dst], env=env, capture_output=True,
                       text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    want, status, lib = run_cases()
    assert status == 0 and lib.endswith("libinkling_fa4.so")
    got = torch.load(dst)
    assert got["lib"].endswith("libinkling_fa4_debug.so") and got["status"] == 0
    assert got["outs"].keys() == want.keys()
    for k, v in want.items():
        torch.testing.assert_close(got["outs"][k], v, atol=0, rtol=0, equal_nan=True, msg=k)


if __name__ == "__main__":
    o, s, p = run_cases()
    torch.save(dict(outs=o, status=s, lib=p), sys.argv[1])
