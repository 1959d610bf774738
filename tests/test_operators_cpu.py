"""What of the operators next to the attention needs no GPU: the ctypes mirrors of their parameter
blocks, the refusals of the C ABI (before any CUDA call), the refusals of the Python entry points
for CPU tensors, the bucket starts, and the oracle's gradients against differences."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

import oracle
from conftest import REPO
from inkling_fa4 import (_lib, inkling_bucket_bias, inkling_bucket_bias_backward,
                         inkling_fa4_rel_attention_decode_shared_prefix, inkling_kv_append,
                         inkling_qk_norm_rope, inkling_qk_norm_rope_backward,
                         relative_bucket_starts)

INVALID, UNSUPPORTED = _lib.IFA4_ERR_INVALID_ARGUMENT, _lib.IFA4_ERR_UNSUPPORTED
HEADER_DIR = os.path.join(REPO, "include")


@pytest.mark.parametrize("cls,cname", [
    (_lib.SharedPrefixParams, "IFA4SharedPrefixParams"),
    (_lib.QkNormRopeParams, "IFA4QkNormRopeParams"),
    (_lib.QkNormRopeBackwardParams, "IFA4QkNormRopeBackwardParams"),
    (_lib.KvAppendParams, "IFA4KvAppendParams"),
    (_lib.BucketBiasParams, "IFA4BucketBiasParams"),
    (_lib.BucketBiasBackwardParams, "IFA4BucketBiasBackwardParams")])
def test_struct_layout_matches_header(cls, cname):
    fields = [f[0] for f in cls._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"inkling_fa4.h\"\nint main(){\n"
    src += f'printf("%zu\\n", sizeof({cname}));\n'
    src += "".join(f'printf("%zu\\n", offsetof({cname}, {f}));\n' for f in fields)
    src += "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", HEADER_DIR, c, "-o", exe], check=True)
        vals = [int(x) for x in subprocess.run([exe], capture_output=True, text=True,
                                               check=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(cls)
    assert vals[1:] == [getattr(cls, f).offset for f in fields]


def _refused(fn, p, code, msg, *rest):
    rc = getattr(_lib.lib(), fn)(ctypes.byref(p), *rest)
    text = _lib.lib().ifa4_last_error_string()
    assert rc == code and msg in text, (rc, text)


def _set(p, **kw):
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _norm_rope(**kw):
    p = _set(_lib.QkNormRopeParams(), q=256, k=256, q_out=256, k_out=256, total_q=4, batch=1,
             n_heads=4, kv_heads=2, head_dim=128, rotary_dim=64, inv_freq=256, normalize=1,
             eps=1e-6)
    for nm in ("q", "k", "q_out", "k_out"):
        _set(p, **{f"{nm}_stride_t": 512, f"{nm}_stride_h": 128})
    return _set(p, **kw)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(head_dim=64), UNSUPPORTED, b"head_dim"),
    (dict(dtype=2), UNSUPPORTED, b"dtype"),
    (dict(rotary_dim=24), UNSUPPORTED, b"rotary_dim"),
    (dict(rotary_dim=144), UNSUPPORTED, b"rotary_dim"),
    (dict(rotary_dim=-16), UNSUPPORTED, b"rotary_dim"),
    (dict(inv_freq=None), INVALID, b"inv_freq"),
    (dict(inv_freq=260), INVALID, b"inv_freq"),
    (dict(weight_dtype=5), UNSUPPORTED, b"weight_dtype"),
    (dict(q_weight=255), INVALID, b"weights"),
    (dict(normalize=0, k_weight=256), INVALID, b"without the norm"),
    (dict(eps=-1.0), INVALID, b"eps"),
    (dict(eps=float("nan")), INVALID, b"eps"),
    (dict(cu_seqlens_k=256), INVALID, b"cu_seqlens_k"),
    (dict(cu_seqlens_q=256, batch=0), INVALID, b"batch"),
    (dict(total_q=-1), INVALID, b"total_q"),
    (dict(n_heads=-1), INVALID, b"head counts"),
    (dict(q=None), INVALID, b"q is NULL"),
    (dict(k_out=264), INVALID, b"16-byte"),
    (dict(q_stride_t=516), INVALID, b"multiples of 8"),
    (dict(q_out_stride_t=0), INVALID, b"positive"),
])
def test_norm_rope_refusals(kw, code, msg):
    _refused("ifa4_qk_norm_rope_launch", _norm_rope(**kw), code, msg, None)


def test_empty_calls_are_no_ops():
    L = _lib.lib()
    assert L.ifa4_qk_norm_rope_launch(ctypes.byref(_norm_rope(total_q=0)), None) == 0
    assert L.ifa4_kv_append_launch(ctypes.byref(_append(total_q=0)), None) == 0
    assert L.ifa4_decode_shared_prefix_launch(ctypes.byref(_shared(total_q=0, batch=0)), None, 0,
                                              None) == 0


def _backward(**kw):
    p = _set(_lib.QkNormRopeBackwardParams(), total_q=4, batch=1, n_heads=4, kv_heads=2,
             head_dim=128, normalize=1, eps=1e-6)
    for nm in ("dq_out", "dk_out", "q", "k", "dq", "dk"):
        _set(p, **{nm: 256, f"{nm}_stride_t": 512, f"{nm}_stride_h": 128})
    return _set(p, **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(dq_out=None), b"dq_out is NULL"), (dict(dk=264), b"16-byte"),
    (dict(dq_stride_h=0), b"positive"), (dict(normalize=0, dq_weight=256), b"without the norm"),
    (dict(dk_weight=255), b"misaligned"),
])
def test_norm_rope_backward_refusals(kw, msg):
    _refused("ifa4_qk_norm_rope_backward_launch", _backward(**kw), INVALID, msg, None, 0, None)
    nbytes = ctypes.c_size_t(0)
    _refused("ifa4_qk_norm_rope_backward_workspace_size", _backward(**kw), INVALID, msg,
             ctypes.byref(nbytes))


def _append(**kw):
    p = _set(_lib.KvAppendParams(), total_q=4, batch=2, n_heads=0, kv_heads=2, head_dim=128,
             normalize=1, eps=1e-6, page_size=16, num_pages=8, table_width=3,
             block_table=256, block_table_stride=3, cu_seqlens_q=256, cu_seqlens_k=256,
             k_cache=256, v_cache=512, k_stride_page=4096, k_cache_stride_t=256,
             k_cache_stride_h=128, v_stride_page=4096, v_cache_stride_t=256, v_cache_stride_h=128)
    for nm in ("k", "v"):
        _set(p, **{nm: 256, f"{nm}_stride_t": 512, f"{nm}_stride_h": 128})
    return _set(p, **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(page_size=8), b"page_size"), (dict(page_size=48), b"page_size"),
    (dict(num_pages=-1), b"negative"), (dict(block_table_stride=-1), b"negative"),
    (dict(kv_heads=0), b"kv_heads"), (dict(block_table=None), b"block_table"),
    (dict(cu_seqlens_k=None), b"cu_seqlens_k"), (dict(n_heads=4), b"q is NULL"),
    (dict(v=None), b"v is NULL"), (dict(k_cache=260), b"16-byte"),
    (dict(k_stride_page=100), b"page strides"), (dict(v_cache_stride_h=4), b"multiples of 8"),
])
def test_kv_append_refusals(kw, msg):
    _refused("ifa4_kv_append_launch", _append(**kw), INVALID, msg, None)


def _shared(**kw):
    p = _lib.SharedPrefixParams()
    d = _set(p.decode, q=256, k=256, v=256, rel=256, out=256, cu_seqlens_q=256, cu_seqlens_k=256,
             batch=2, total_q=2, total_k=64, n_heads=4, kv_heads=2, head_dim=128, rel_extent=16,
             causal=1, window_left=-1, causal_align=_lib.IFA4_ALIGN_BOTTOM_RIGHT,
             softmax_scale=0.1, block_table=256, block_table_stride=4, page_size=16, num_pages=4,
             k_stride_page=4096, v_stride_page=4096)
    for nm in ("q", "k", "v", "rel", "out"):
        _set(d, **{f"{nm}_stride_t": 512, f"{nm}_stride_h": 128})
    p.shared_prefix_len = 32
    for k, v in kw.items():
        setattr(p if k in ("shared_prefix_len", "prefix_splits") else d, k, v)
    return p


@pytest.mark.parametrize("kw,code,msg", [
    (dict(shared_prefix_len=-1), INVALID, b"shared_prefix_len"),
    (dict(shared_prefix_len=(1 << 30) + 1), INVALID, b"shared_prefix_len"),
    (dict(prefix_splits=-1), INVALID, b"prefix_splits"),
    (dict(block_table=None), INVALID, b"block_table"),
    (dict(causal_align=_lib.IFA4_ALIGN_REFERENCE), UNSUPPORTED, b"bottom-right"),
    (dict(n_heads=258, kv_heads=2), UNSUPPORTED, b"128 query heads"),
    (dict(total_q=3), INVALID, b"one query"),
    (dict(page_size=24), INVALID, b"page_size"),
    (dict(chunk_len=10), INVALID, b"chunk_len"),
])
def test_shared_prefix_refusals(kw, code, msg):
    _refused("ifa4_decode_shared_prefix_launch", _shared(**kw), code, msg, None, 0, None)


def test_shared_prefix_needs_its_workspace():
    # explicit splits and chunk: the plan needs no GPU
    p = _shared(prefix_splits=2, num_splits=3, chunk_len=64)
    nbytes = ctypes.c_size_t(0)
    L = _lib.lib()
    rc = L.ifa4_decode_shared_prefix_workspace_size(ctypes.byref(p), ctypes.byref(nbytes))
    if rc == _lib.IFA4_ERR_CUDA:
        pytest.skip("the plan asked the CUDA runtime for the SM count")
    assert rc == 0
    assert nbytes.value == 2 * 4 * (2 * 2 + 3) * 129 * 4  # one row tile: two partials a split
    _refused("ifa4_decode_shared_prefix_launch", p, _lib.IFA4_ERR_WORKSPACE, b"workspace", None, 0,
             None)


def _bucket(**kw):
    return _set(_set(_lib.BucketBiasParams(), table=256, starts=256, rel=256, table_stride_b=4,
                     table_stride_h=1, rel_stride_h=16, n_heads=4, rel_extent=16, buckets=8), **kw)


def _bucket_backward(**kw):
    return _set(_set(_lib.BucketBiasBackwardParams(), drel=256, starts=256, dtable=256,
                     drel_stride_t=64, drel_stride_h=16, dtable_stride_b=4, dtable_stride_h=1,
                     total_q=8, n_heads=4, rel_extent=16, buckets=8), **kw)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(n_heads=0), INVALID, b"n_heads"), (dict(rel_extent=0), INVALID, b"rel_extent"),
    (dict(buckets=0), INVALID, b"buckets"), (dict(buckets=1025), INVALID, b"buckets"),
    (dict(weight_dtype=9), UNSUPPORTED, b"weight_dtype"), (dict(starts=None), INVALID, b"starts"),
])
def test_bucket_refusals(kw, code, msg):
    _refused("ifa4_bucket_bias_launch", _bucket(**kw), code, msg, None)
    _refused("ifa4_bucket_bias_backward_launch", _bucket_backward(**kw), code, msg, None, 0, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(drel=None), b"drel"), (dict(dtable=None), b"dtable"), (dict(total_q=-1), b"total_q"),
    (dict(drel_stride_t=-8), b"strides"), (dict(drel=257), b"misaligned"),
])
def test_bucket_backward_refusals(kw, msg):
    _refused("ifa4_bucket_bias_backward_launch", _bucket_backward(**kw), INVALID, msg, None, 0,
             None)


def test_python_entry_points_refuse_cpu_tensors():
    x = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 2], dtype=torch.int32)
    cache = torch.zeros(2, 16, 4, 128, dtype=torch.bfloat16)
    table = torch.zeros(1, 2, dtype=torch.int32)
    rel = torch.zeros(2, 4, 16, dtype=torch.bfloat16)
    starts = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: inkling_qk_norm_rope(x, x),
                 lambda: inkling_qk_norm_rope_backward(x, x, x, x),
                 lambda: inkling_kv_append(x, x, cache, cache.clone(), table, cu, cu),
                 lambda: inkling_fa4_rel_attention_decode_shared_prefix(
                     x, cache, cache, rel, cu, cu, 1, 32, 16, 16, block_table=table),
                 lambda: inkling_bucket_bias(torch.zeros(1, 4), starts, 2, 16),
                 lambda: inkling_bucket_bias_backward(rel, starts, 1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_bucket_starts():
    assert relative_bucket_starts(32, 128) == list(range(17)) + [19, 21, 24, 27, 31, 35, 40, 46, 52,
                                                                 59, 67, 77, 87, 99, 113]
    # exact powers sit on the border: 16 * 64^(8/16) = 128 begins its bucket
    assert relative_bucket_starts(32, 1024)[24] == 128
    assert relative_bucket_starts(8, 1024) == [0, 1, 2, 3, 4, 16, 64, 256]
    for nb, md in ((2, 2), (3, 7), (9, 100), (64, 64), (1024, 1024), (256, 100000)):
        s = relative_bucket_starts(nb, md)
        e, n = nb // 2, nb - nb // 2
        assert len(s) == nb and s[0] == 0 and s == sorted(s) and s[-1] <= md
        for j in range(n):
            want = md ** j * e ** (n - j)
            assert s[e + j] ** n >= want and (s[e + j] - 1) ** n < want
    with pytest.raises(ValueError):
        relative_bucket_starts(1, 10)
    with pytest.raises(ValueError):
        relative_bucket_starts(64, 63)
    with pytest.raises(ValueError):
        relative_bucket_starts(2000, 5000)


@pytest.mark.parametrize("rot,interleaved,eps", [(0, False, 1e-3), (64, False, 1e-3),
                                                 (128, True, 1e-3), (96, True, None)])
def test_oracle_gradient_against_differences(rot, interleaved, eps):
    """Central differences of the oracle's forward: the step 1e-5 leaves about 1e-10 of truncation
    and 1e-11 of rounding in 64 bits; 1e-7 bounds both."""
    rng = np.random.default_rng(3)
    x, w, g = rng.normal(size=(3, 2, 128)), rng.normal(size=128) + 1, rng.normal(size=(3, 2, 128))
    inv = None if rot == 0 else 100.0 ** (-np.arange(rot // 2) / (rot / 2))
    pos = np.array([0, 5, 77])
    w = None if eps is None else w

    def loss(x, w):
        return (oracle.norm_rope(x, w, pos, eps, inv, interleaved) * g).sum()

    dx, dw, _, _ = oracle.norm_rope_grads(g, x, w, pos, eps, inv, interleaved)
    h = 1e-5
    for _ in range(20):
        i = tuple(rng.integers(n) for n in x.shape)
        step = np.zeros_like(x)
        step[i] = h
        assert abs((loss(x + step, w) - loss(x - step, w)) / (2 * h) - dx[i]) < 1e-7
        if w is not None:
            j = rng.integers(128)
            step = np.zeros_like(w)
            step[j] = h
            assert abs((loss(x, w + step) - loss(x, w - step)) / (2 * h) - dw[j]) < 1e-7


def test_plain_calls():
    """Every Python call of the operator library is there; what is not its plain case (the wrong
    number or types of arguments, tensors on the CPU) gives None, not an error."""
    assert _lib.torch_ops() is not None, "libifa4_torch_ops.so not built"
    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    norm = (x, x, None, None, None, None, None, False, 1e-6)
    calls = {"decode_shared_prefix": (), "qk_norm_rope": norm, "kv_append": (x,) * 15,
             "qk_norm_rope_backward": (x, x, *norm, True, True),
             "bucket_bias": (x[0], torch.zeros(2, dtype=torch.int32), 4, 16),
             "bucket_bias_backward": (x, torch.zeros(2, dtype=torch.int32), True, None)}
    for name, args in calls.items():
        assert name in _lib._calls
        for a in (args, (), args + (None,), args[:-1] + (object(),), (None,) * len(args),
                  (1 << 70,) * len(args)):
            assert _lib.plain_call(name, *a) is None, (name, a)
