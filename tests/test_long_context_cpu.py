"""What of the long-context operators needs no GPU: the ctypes mirrors of their parameter blocks, the
refusals of the C ABI (before any CUDA call), the refusals of the Python entry points, and the
oracle's choice of the largest against a sort."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

import inkling_fa4
from conftest import REPO
from inkling_fa4 import _lib, _paged
from oracle import long_context_oracle as oracle

INVALID, UNSUPPORTED = _lib.IFA4_ERR_INVALID_ARGUMENT, _lib.IFA4_ERR_UNSUPPORTED
WORKSPACE = _lib.IFA4_ERR_WORKSPACE


@pytest.mark.parametrize("name", ["PagedSeqs", "PageBoundsParams", "PageScoresParams",
                                  "SelectPagesParams", "DecodePagesParams", "AttentionMassParams",
                                  "KvEvictParams"])
def test_struct_layout_matches_header(name):
    cls = getattr(_lib, name)
    fields = [f[0] for f in cls._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"inkling_fa4.h\"\nint main(){\n"
    src += f'printf("%zu\\n", sizeof(IFA4{name}));\n'
    src += "".join(f'printf("%zu\\n", offsetof(IFA4{name}, {f}));\n' for f in fields)
    src += "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), c, "-o", exe], check=True)
        vals = [int(x) for x in subprocess.run([exe], capture_output=True, text=True,
                                               check=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(cls)
    assert vals[1:] == [getattr(cls, f).offset for f in fields]


def _set(p, **kw):
    for k, v in kw.items():
        if k in ("batch", "page_size", "num_pages", "table_width", "block_table", "cu_seqlens_q",
                 "cu_seqlens_k", "block_table_stride") and hasattr(p, "seqs"):
            setattr(p.seqs, k, v)
        elif hasattr(p, "decode") and not hasattr(type(p), k):
            setattr(p.decode, k, v)
        else:
            setattr(p, k, v)
    return p


SEQS = dict(batch=2, page_size=16, num_pages=8, table_width=4, block_table=256, cu_seqlens_q=256,
            cu_seqlens_k=256, block_table_stride=4)
CACHE = dict(k_cache=256, k_stride_page=4096, k_stride_t=256, k_stride_h=128, kv_heads=2,
             head_dim=128)
BOUNDS = dict(bounds=256, bounds_stride_page=512, bounds_stride_h=256)
QUERY = dict(q=256, q_stride_t=512, q_stride_h=128, rel=256, rel_stride_t=64, rel_stride_h=16,
             total_q=2, n_heads=4, rel_extent=16, softmax_scale=1.0)
COMMON = [(dict(page_size=24), INVALID, b"page_size"), (dict(page_size=8), INVALID, b"page_size"),
          (dict(batch=-1), INVALID, b"batch"), (dict(batch=65535), UNSUPPORTED, b"batch"),
          (dict(num_pages=-1), INVALID, b"num_pages"), (dict(table_width=-1), INVALID, b"table_width"),
          (dict(table_width=(1 << 26) + 1), UNSUPPORTED, b"table_width"),
          (dict(block_table=None), INVALID, b"block_table"),
          (dict(cu_seqlens_k=None), INVALID, b"cu_seqlens"),
          (dict(head_dim=64), UNSUPPORTED, b"head_dim"), (dict(dtype=1), UNSUPPORTED, b"dtype"),
          (dict(kv_heads=0), INVALID, b"kv_heads")]
KEYS = [(dict(k_cache=264), INVALID, b"k_cache"), (dict(k_cache=None), INVALID, b"k_cache"),
        (dict(k_stride_t=100), INVALID, b"k_cache"), (dict(k_stride_page=0), INVALID, b"k_cache")]
QUERIES = [(dict(q=None), INVALID, b"null"), (dict(q_stride_t=0), INVALID, b"q needs"),
           (dict(q=260), INVALID, b"q needs"), (dict(rel_extent=0), INVALID, b"rel_extent"),
           (dict(softmax_scale=0.0), INVALID, b"softmax_scale"),
           (dict(softmax_scale=float("nan")), INVALID, b"softmax_scale"),
           (dict(softmax_scale=float("inf")), INVALID, b"softmax_scale"),
           (dict(rel=257), INVALID, b"misaligned rel"), (dict(cu_seqlens_q=258), INVALID, b"cu_seqlens"),
           (dict(rel_stride_t=-1), INVALID, b"rel"), (dict(total_q=-1), INVALID, b"total_q"),
           (dict(n_heads=5), INVALID, b"n_heads")]


def _refused(fn, p, code, msg, *rest):
    rc = getattr(_lib.lib(), fn)(ctypes.byref(p), *rest)
    text = _lib.lib().ifa4_last_error_string()
    assert rc == code and msg in text, (rc, text)


@pytest.mark.parametrize("kw,code,msg", COMMON + KEYS + [
    (dict(bounds=None), INVALID, b"bounds"), (dict(bounds_stride_page=0), INVALID, b"bounds"),
    (dict(bounds_stride_h=128), INVALID, b"overlap"), (dict(bounds_stride_page=256), INVALID, b"overlap"),
    (dict(block_table=257), INVALID, b"misaligned"), (dict(cu_seqlens_k=258), INVALID, b"misaligned"),
    (dict(cu_seqlens_q=None), INVALID, b"cu_seqlens")])
def test_page_bounds_refusals(kw, code, msg):
    _refused("ifa4_page_bounds_launch", _set(_lib.PageBoundsParams(), **{**SEQS, **CACHE, **BOUNDS, **kw}),
             code, msg, None)


@pytest.mark.parametrize("kw,code,msg", [x for x in COMMON if x[2] != b"kv_heads"] + QUERIES + [
    (dict(bounds=None), INVALID, b"bounds"), (dict(first_pages=-1), INVALID, b"first_pages"),
    (dict(scores=None), INVALID, b"scores"), (dict(scores_stride_t=-1), INVALID, b"strides"),
    (dict(scores=258), INVALID, b"misaligned"), (dict(scores_stride_h=3), INVALID, b"overlap"),
    (dict(scores_stride_t=0), INVALID, b"overlap")])
def test_page_scores_refusals(kw, code, msg):
    base = {**SEQS, **BOUNDS, **QUERY, "kv_heads": 2, "head_dim": 128, "scores": 256,
            "scores_stride_t": 8, "scores_stride_h": 4}
    _refused("ifa4_page_scores_launch", _set(_lib.PageScoresParams(), **{**base, **kw}), code, msg, None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(num_selected=0), INVALID, b"num_selected"), (dict(width=-1), INVALID, b"width"),
    (dict(rows=-1), INVALID, b"rows"), (dict(scores=None), INVALID, b"null"),
    (dict(pages=None), INVALID, b"null"), (dict(pages_stride_h=-1), INVALID, b"strides"),
    (dict(scores=258), INVALID, b"misaligned"), (dict(pages=257), INVALID, b"misaligned"),
    (dict(pages_stride_t=2), INVALID, b"overlap"), (dict(kv_heads=65536), INVALID, b"kv_heads")])
def test_select_pages_refusals(kw, code, msg):
    base = dict(scores=256, pages=256, rows=2, kv_heads=2, width=4, num_selected=2, pages_stride_t=4,
                pages_stride_h=2)
    _refused("ifa4_select_pages_launch", _set(_lib.SelectPagesParams(), **{**base, **kw}), code, msg, None)


def _decode_pages(**kw):
    p = _lib.DecodePagesParams()
    base = dict(q=256, k=256, v=256, rel=256, out=256, cu_seqlens_q=256, cu_seqlens_k=256,
                block_table=256, q_stride_t=512, q_stride_h=128, k_stride_t=256, k_stride_h=128,
                v_stride_t=256, v_stride_h=128, k_stride_page=4096, v_stride_page=4096,
                rel_stride_t=64, rel_stride_h=16, out_stride_t=512, out_stride_h=128, total_q=3,
                batch=2, n_heads=4, kv_heads=2, head_dim=128, rel_extent=16, causal=1, window_left=-1,
                causal_align=1, page_size=16, num_pages=8, softmax_scale=1.0, num_splits=2)
    own = dict(pages=256, num_selected=4, table_width=4)
    for k, v in {**base, **own, **kw}.items():
        setattr(p if k in ("pages", "num_selected", "table_width", "pages_stride_t") else p.decode, k, v)
    return p


@pytest.mark.parametrize("kw,code,msg", [
    (dict(block_table=None), INVALID, b"block_table"), (dict(causal=0), INVALID, b"causal"),
    (dict(causal_align=0), INVALID, b"BOTTOM_RIGHT"), (dict(pages=None), INVALID, b"pages"),
    (dict(num_selected=-1), INVALID, b"num_selected"), (dict(num_splits=-1), INVALID, b"num_splits"),
    (dict(num_splits=1025), INVALID, b"num_splits"),
    (dict(num_selected=1 << 26, page_size=1 << 12), UNSUPPORTED, b"2^36"),
    (dict(page_size=24), INVALID, b"page_size"),
    (dict(total_q=1 << 31), UNSUPPORTED, b"rows"), (dict(batch=65535), UNSUPPORTED, b"batch"),
    (dict(pages=258), INVALID, b"misaligned"), (dict(rel=257), INVALID, b"misaligned"),
    (dict(lse=258), INVALID, b"misaligned"), (dict(block_table=257), INVALID, b"misaligned"),
    (dict(softmax_scale=float("inf")), INVALID, b"softmax_scale"),
    (dict(q=260), INVALID, b"aligned")])
def test_decode_pages_refusals(kw, code, msg):
    need = ctypes.c_size_t(0)
    _refused("ifa4_decode_pages_workspace_size", _decode_pages(**kw), code, msg, ctypes.byref(need))
    _refused("ifa4_decode_pages_launch", _decode_pages(**kw), code, msg, None, ctypes.c_size_t(0), None)


def test_decode_pages_workspace():
    need = ctypes.c_size_t(0)
    L = _lib.lib()
    for splits, want in ((1, 0), (8, 0), (9, 3 * 4 * 9 * 130 * 4), (64, 3 * 4 * 64 * 130 * 4)):
        assert L.ifa4_decode_pages_workspace_size(ctypes.byref(_decode_pages(num_splits=splits)),
                                                  ctypes.byref(need)) == 0
        assert need.value == want
    many = _decode_pages(num_splits=9)
    _refused("ifa4_decode_pages_launch", many, WORKSPACE, b"workspace", None, ctypes.c_size_t(0), None)
    _refused("ifa4_decode_pages_launch", many, WORKSPACE, b"aligned", ctypes.c_void_p(264),
             ctypes.c_size_t(1 << 20), None)


@pytest.mark.parametrize("kw,code,msg", COMMON[:-1] + KEYS + QUERIES + [
    (dict(n_heads=258), UNSUPPORTED, b"128"), (dict(mass_width=-1), INVALID, b"mass_width"),
    (dict(mass=None), INVALID, b"null"), (dict(lse=None), INVALID, b"null"),
    (dict(mass_stride_b=-1), INVALID, b"mass"), (dict(num_pages=0), INVALID, b"num_pages"),
    (dict(mass=258), INVALID, b"misaligned"), (dict(lse=257), INVALID, b"misaligned"),
    (dict(mass_stride_h=63), INVALID, b"overlap"), (dict(mass_stride_b=0), INVALID, b"overlap")])
def test_attention_mass_refusals(kw, code, msg):
    base = {**SEQS, **CACHE, **QUERY, "lse": 256, "mass": 256, "mass_width": 64, "mass_stride_b": 128,
            "mass_stride_h": 64}
    _refused("ifa4_attention_mass_launch", _set(_lib.AttentionMassParams(), **{**base, **kw}), code, msg,
             None)


@pytest.mark.parametrize("kw,code,msg", COMMON + KEYS + [
    (dict(v_cache=264), INVALID, b"v_cache"), (dict(budget=0), INVALID, b"budget"),
    (dict(first=3, recent=2), INVALID, b"budget"), (dict(first=-1), INVALID, b"budget"),
    (dict(mass=None), INVALID, b"null"), (dict(mass=512), INVALID, b"mass_out"),
    (dict(kept=None), INVALID, b"null"), (dict(cu_out=None), INVALID, b"cu_out"),
    (dict(kept=258), INVALID, b"misaligned"), (dict(cu_out=257), INVALID, b"misaligned"),
    (dict(k_stride_t=128), INVALID, b"overlap"), (dict(v_stride_page=2048), INVALID, b"overlap"),
    (dict(mass_stride_b=-1), INVALID, b"mass"), (dict(mass_out_stride_h=0), INVALID, b"overlap"),
    (dict(mass_width=-1), INVALID, b"mass_width")])
def test_kv_evict_refusals(kw, code, msg):
    base = {**SEQS, **CACHE, "v_cache": 512, "v_stride_page": 4096, "v_stride_t": 256,
            "v_stride_h": 128, "mass": 256, "mass_out": 512, "kept": 256, "cu_out": 256,
            "mass_width": 64, "mass_stride_b": 128, "mass_stride_h": 64, "mass_out_stride_b": 128,
            "mass_out_stride_h": 64, "budget": 4}
    need = ctypes.c_size_t(0)
    p = _set(_lib.KvEvictParams(), **{**base, **kw})
    _refused("ifa4_kv_evict_workspace_size", p, code, msg, ctypes.byref(need))
    _refused("ifa4_kv_evict_launch", p, code, msg, None, ctypes.c_size_t(0), None)


@pytest.mark.parametrize("name", ["page_bounds", "page_scores", "select_pages", "attention_mass"])
def test_null_params_are_refused(name):
    assert getattr(_lib.lib(), f"ifa4_{name}_launch")(None, None) == INVALID
    assert b"NULL" in _lib.lib().ifa4_last_error_string()


def _cpu():
    bf16, i32 = torch.bfloat16, torch.int32
    return dict(k=torch.zeros(2, 16, 1, 128, dtype=bf16), bounds=torch.zeros(2, 1, 2, 128, dtype=bf16),
                q=torch.zeros(1, 1, 128, dtype=bf16), rel=torch.zeros(1, 1, 8, dtype=bf16),
                table=torch.zeros(1, 2, dtype=i32), cu=torch.tensor([0, 1], dtype=i32),
                pages=torch.zeros(1, 1, 1, dtype=i32), lse=torch.zeros(1, 1), mass=torch.zeros(1, 1, 32))


def test_cpu_tensors_are_refused():
    c = _cpu()
    calls = [
        lambda: inkling_fa4.inkling_kv_page_bounds(c["k"], c["table"], c["cu"], c["cu"]),
        lambda: inkling_fa4.inkling_kv_page_bounds(c["k"], c["table"], c["cu"], c["cu"], 1,
                                                   bounds=c["bounds"]),
        lambda: inkling_fa4.inkling_kv_page_scores(c["q"], c["bounds"], c["rel"], c["cu"], c["cu"], 1, 8,
                                                   16, block_table=c["table"]),
        lambda: inkling_fa4.inkling_kv_select_pages(torch.zeros(1, 1, 4), 2),
        lambda: inkling_fa4.inkling_fa4_rel_attention_decode_pages(
            c["q"], c["k"], c["k"].clone(), c["rel"], c["cu"], c["cu"], 1, 1, 8, c["pages"],
            block_table=c["table"]),
        lambda: inkling_fa4.inkling_kv_attention_mass(c["q"], c["k"], c["rel"], c["lse"], c["cu"],
                                                      c["cu"], 1, 1, 8, block_table=c["table"]),
        lambda: inkling_fa4.inkling_kv_evict(c["k"], c["k"].clone(), c["mass"], c["table"], c["cu"], 4)]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_things_that_are_no_tensors_are_refused():
    with pytest.raises(TypeError, match="torch.Tensor"):
        inkling_fa4.inkling_kv_select_pages([1.0], 2)
    with pytest.raises(TypeError, match="torch.Tensor"):
        inkling_fa4.inkling_kv_evict(None, None, None, None, None, 4)


def test_rows_apart():
    """Against the sets of elements."""
    base = torch.zeros(4000)
    for shape in ((2, 3, 4), (1, 3, 4), (3, 1, 5), (1, 1, 7), (2, 2, 1)):
        for st in (0, 1, 4, 5, 8, 12, 15, 20):
            for sh in (0, 1, 3, 4, 5, 8, 16):
                t = base.as_strided(shape, (st, sh, 1))
                seen = set()
                rows = [{t[i, j].storage_offset() + k for k in range(shape[2])}
                        for i in range(shape[0]) for j in range(shape[1])]
                apart = sum(map(len, rows)) == len(set().union(*rows))
                if _paged.rows_apart(t):
                    assert apart, (shape, st, sh)
                elif apart:  # what is refused and need not be: rows that lie between other rows
                    assert min(shape[:2]) > 1, (shape, st, sh)


@pytest.mark.parametrize("seed", range(5))
def test_oracle_choice(seed):
    rng = np.random.default_rng(seed)
    x = np.round(rng.standard_normal(60) * 2) / 2
    x[rng.integers(0, 60, 5)] = -np.inf
    got = oracle.select_largest(x, 20)
    order = np.argsort(-x, kind="stable")
    assert got == sorted(i for i in order[:20] if x[i] > -np.inf)
