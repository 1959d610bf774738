"""The index checks of the long-context kernels can fail: in the debug build, offsets that name more rows
than a call has (or rows in front of them) are reported in the status word, and the rows behind (in front)
are neither read for an output nor written.  Every tensor is a slice of a larger one, so that the rows
that the offsets name exist whatever the kernels do; each call has one sequence, so that nothing waits
while the status word is set."""
import os
import subprocess
import sys

import pytest
import torch

from inkling_fa4 import _lib, inkling_kv_attention_mass, inkling_kv_page_bounds, inkling_kv_page_scores
from long_context_cases import Case

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
DEBUG_LIB = os.path.join(os.path.dirname(_lib.LIB_PATH), "libinkling_fa4_debug.so")
FAILED = 64


def run_cases():
    c = Case([64], [200], 8, 2, 16, 50, seed=81)
    bounds = inkling_kv_page_bounds(c.k, c.table, c.cu_k, c.cu_k)
    seen = {}

    def status():
        return _lib.read_device_status(torch.cuda.current_stream().cuda_stream, clear=True)

    assert status() == 0
    for name, ends in (("as many as there are", (0, 10)), ("more than there are", (0, 40)),
                       ("in front", (-3, 7))):
        cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
        rows = slice(20, 30)
        q, rel = c.q[rows], c.rel[rows]
        scores = torch.full((64, 2, c.width), 3.0, device="cuda")
        inkling_kv_page_scores(q, bounds, rel, cu, c.cu_k, 10, 50, 16, block_table=c.table,
                               out=scores[rows])
        code = status()
        scores[rows] = 3.0
        seen[f"scores, {name}"] = code, not bool((scores != 3.0).any())
        lse = torch.full((8, 64), 5.0, device="cuda")[:, rows]
        for kernel, hint in (("few rows", 1), ("many rows", 10)):
            mass = torch.zeros(1, 2, c.width * 16, device="cuda")
            inkling_kv_attention_mass(q, c.k, rel, lse, cu, c.cu_k, hint, 200, 50, block_table=c.table,
                                      mass=mass)
            code = status()
            seen[f"mass, {kernel}, {name}"] = code, bool(mass.any()) == (code == 0)
    return seen, _lib.LIB_PATH


@pytest.mark.skipif(not os.path.exists(DEBUG_LIB), reason="debug build not built")
def test_offsets_past_the_rows_are_reported():
    path = os.pathsep.join([HERE, os.path.dirname(os.path.dirname(os.path.dirname(_lib.LIB_PATH)))])
    env = dict(os.environ, INKLING_FA4_LIB="debug", PYTHONPATH=path)
    r = subprocess.run([sys.executable, os.path.abspath(__file__)], env=env, capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = r.stdout.strip().splitlines()
    assert lines[0].endswith("libinkling_fa4_debug.so") and len(lines) == 10
    for line in lines[1:]:
        name, code, kept = line.split(": ")
        want = 0 if name.endswith("as many as there are") else FAILED
        assert int(code) == want and kept == "True", line


if __name__ == "__main__":
    result, lib = run_cases()
    print(lib)
    for key, (code, kept) in result.items():
        print(f"{key}: {code}: {kept}")
