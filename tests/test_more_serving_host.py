"""Quantised caches, norms and rotation, and attention with shared prefixes without a
GPU: refusals of the C ABI and of the Python layer, and the oracle's own invariants."""
import ctypes
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from llm_gpu_kernels_amd import (PagedKVCache, _native as N, prepare_paged_gqa, prepare_qk_norm_rope,
                                 prepare_shared_gqa)
from oracle import serving_oracle as S

ROOT = Path(__file__).resolve().parents[1]
BASE = 1 << 20  # an address that is only looked at by the validation


def _cache_desc():
    d = N.KvCacheDesc()
    d.pages, d.page_size, d.kv_heads, d.head_dim, d.layers = 100, 16, 8, 128, 2
    d.sequences, d.max_pages, d.max_tokens = 4, 10, 64
    for name in ("k", "v", "tables", "lengths", "refs", "starts", "slots", "status", "workspace"):
        setattr(d, name, BASE)
    d.workspace_bytes = 1 << 30
    return d


@pytest.mark.parametrize("storage,tokens,ks,vs", [(3, 0, BASE, BASE), (-1, 0, None, None), (1, 2, BASE, BASE), (1, 0, None, BASE),
                                                  (1, 0, BASE, BASE + 8), (2, 1, BASE, None), (0, 0, BASE, BASE)])
def test_stored_cache_refusals(storage, tokens, ks, vs):
    handle = ctypes.c_void_p()
    rc = N.lib().kv_cache_create_stored(ctypes.byref(handle), ctypes.byref(_cache_desc()), storage, tokens, ks, vs)
    assert rc == N.MOE_EINVAL and not handle.value and N.last_error()


def test_gather_null():
    assert N.lib().kv_cache_gather(None, 0, BASE, BASE, 1, BASE, BASE, 1024, 1024, 5, None) == N.MOE_EINVAL


def test_storage_names():
    good = dict(sequences=4, max_pages=8, max_tokens=64)
    for storage in ("fp8", "mxfp6", 8, "", torch.float8_e4m3fn):
        with pytest.raises(ValueError, match="storage"):
            PagedKVCache(10, 16, 2, 64, storage=storage, **good)


def _qk(**kw):
    d = N.QkNormRopeDesc()
    d.N, d.Hq, d.Hkv, d.D, d.R = 10, 32, 8, 128, 128
    for name in ("q", "k", "positions", "inv_freq", "q_weight", "k_weight", "q_out", "k_out"):
        setattr(d, name, BASE)
    d.q_stride, d.k_stride, d.v_stride, d.eps = 4096, 1024, 1024, 1e-6
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def test_struct_size_matches_header():
    # 8 int32 + 9 pointers + 3 int64 + float + int32.
    assert ctypes.sizeof(N.QkNormRopeDesc) == 32 + 72 + 24 + 8


@pytest.mark.parametrize("bad", [
    dict(D=96), dict(D=256), dict(R=0), dict(R=130), dict(R=63), dict(R=-2), dict(dtype=2), dict(N=-1), dict(N=(1 << 24) + 1),
    dict(Hq=0), dict(Hkv=0), dict(Hq=1 << 20), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(q=None),
    dict(k=BASE + 8), dict(v=BASE), dict(positions=None), dict(inv_freq=BASE + 2), dict(q_weight=BASE + 4),
    dict(k_weight=BASE + 8), dict(q_out=None), dict(k_out=None), dict(k_out=BASE + 8), dict(q_stride=4088),
    dict(k_stride=1028), dict(q_stride=1 << 41),
])
def test_qk_refusals(bad):
    handle = ctypes.c_void_p()
    rc = N.lib().qk_norm_rope_create(ctypes.byref(handle), ctypes.byref(_qk(**bad)), None)
    assert rc == N.MOE_EINVAL and not handle.value and N.last_error()


def test_qk_null():
    handle = ctypes.c_void_p()
    assert N.lib().qk_norm_rope_run(None, None) == N.MOE_EINVAL
    assert N.lib().qk_norm_rope_create(ctypes.byref(handle), None, None) == N.MOE_EINVAL
    assert N.lib().qk_norm_rope_create(None, ctypes.byref(_qk()), None) == N.MOE_EINVAL
    N.lib().qk_norm_rope_destroy(None)


def test_qk_python_refusals():
    q, k = torch.zeros(6, 4, 128, dtype=torch.bfloat16), torch.zeros(6, 2, 128, dtype=torch.bfloat16)
    p, f, w = torch.zeros(6, dtype=torch.int32), torch.ones(64), torch.ones(128)
    for bad in [(q.float(), k, p, f), (q, k, p.long(), f), (q, k, p, f.double()), (q, k, p, f, w.half()),
                (q, k, p, f, w, w.bfloat16())]:
        with pytest.raises(TypeError):
            prepare_qk_norm_rope(*bad)
    for bad in [(q, k[:5], p, f), (q, k, p[:5], f), (q, k, p, torch.ones(65)), (q, k, p, f[:0]), (q, k, p, f[None]),
                (q, k.half(), p, f), (q[..., :64], k, p, f), (q, k, p, f, w[:64]), (q, k, p, torch.ones(128)[::2]),
                (q, k, p, f, None, torch.ones(256)[::2]), (q[:, :, :100], k, p, f), (q, k, p, f)]:  # the last: not on a GPU
        with pytest.raises(ValueError):
            prepare_qk_norm_rope(*bad)
    for eps in (-1e-6, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            prepare_qk_norm_rope(q, k, p, f, eps=eps)


@pytest.mark.parametrize("storage", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantised_rows(storage, dtype):
    """Values are off by half of an element's step, the largest is never cut off where a
    larger scale is left, quantising the values again changes nothing, and they are
    numbers of the tokens' type."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(500, 64, generator=g) * torch.exp2(torch.randint(-6, 6, (500, 1), generator=g).float())
    x = x.to(dtype)
    codes, scales = S.mx_quantise(x, storage, dtype)
    values = S.mx_values(codes, scales, storage)
    scale = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    relative, absolute = (2.0 ** -4, 2.0 ** -10) if storage == "mxfp8" else (2.0 ** -2, 0.25)
    assert ((values - x.double()).abs() <= torch.maximum(relative * x.double().abs(), absolute * scale)).all()
    assert torch.equal(values.to(dtype).double(), values)
    again = S.mx_values(*S.mx_quantise(values.to(dtype), storage, dtype), storage)
    assert torch.equal(again, values)
    assert torch.equal(S.mx_unpack(S.mx_pack(codes, storage), storage), codes)
    if storage == "mxfp8":
        y = (x.double() / scale).float()
        assert torch.equal(y.to(torch.float8_e4m3fn).view(torch.uint8) & 127, codes & 127)


@pytest.mark.parametrize("storage", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantised_tokens_are_numbers_of_their_type(storage, dtype):
    """Every finite token, the smallest too, beside some powers of two as the largest of its
    block."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x)]
    for e in range(-24, 16, 3) if dtype == torch.float16 else (-133, -120, -100, -10, 0, 60, 127):
        top = torch.tensor(2.0, dtype=torch.float64).pow(e)
        y = x[x.double().abs() <= top]
        y = torch.cat([y, torch.zeros(-len(y) % 31, dtype=dtype)]).view(-1, 31)
        rows = torch.cat([y, top.to(dtype).expand(len(y), 1)], 1)
        values = S.mx_values(*S.mx_quantise(rows, storage, dtype), storage)
        assert torch.equal(values.to(dtype).double(), values)


def test_rotation_keeps_lengths():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 2, 64, generator=g)
    f = torch.rand(20, generator=g)
    for interleaved in (False, True):
        y, _ = S.norm_rope(x, torch.arange(4), f, interleaved=interleaved)
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1))
        assert torch.equal(y[..., 40:], x[..., 40:].double()) and torch.equal(y[0], x[0].double())


# ---- attention over quantised pages, and with shared prefixes ---------------------


def _paged(**kw):
    d = N.GqaPagedDesc()
    d.B, d.Hq, d.Hkv, d.D, d.P, d.page, d.M, d.dtype = 5, 32, 8, 128, 100, 16, 20, N.GQA_BF16
    d.q = d.k = d.v = d.out = d.tables = d.lengths = d.workspace = BASE
    d.q_stride, d.table_stride = 4096, 20
    for st in (d.k_strides, d.v_strides):
        st[0], st[1], st[2] = 16 * 8 * 128, 16 * 128, 128
    d.workspace_bytes = 1 << 30
    for name, value in kw.items():
        setattr(d, name, (ctypes.c_int64 * 3)(*value) if name.endswith("strides") else value)
    return d


def _scales(**kw):
    s = N.GqaPagedScales()
    s.storage, s.k, s.v = N.GQA_STORAGE_MXFP8, BASE, BASE
    for st in (s.k_strides, s.v_strides):
        st[0], st[1] = 8 * 64, 64
    for name, value in kw.items():
        setattr(s, name, (ctypes.c_int64 * 2)(*value) if name.endswith("strides") else value)
    return s


@pytest.mark.parametrize("desc,scales", [
    ({}, dict(storage=0)), ({}, dict(storage=3)), ({}, dict(k=None)), ({}, dict(v=BASE + 8)), ({}, dict(k_strides=(512, 60))),
    ({}, dict(v_strides=(0, 64))), (dict(k_strides=(16384, 2048, 256)), {}), (dict(v_strides=(16384, 2040, 128)), {}),
    (dict(k_strides=(8, 2048, 128)), {}), ({}, dict(storage=N.GQA_STORAGE_MXFP4)), (dict(D=96), {}), (dict(page=24), {}),
    (dict(workspace=None), {}), (dict(workspace_bytes=255), {}), (dict(k=BASE + 4), {}), (dict(q_stride=4090), {}),
])
def test_stored_attention_refusals(desc, scales):
    handle = ctypes.c_void_p()
    rc = N.lib().gqa_paged_stored_plan_create(ctypes.byref(handle), ctypes.byref(_paged(**desc)), ctypes.byref(_scales(**scales)))
    assert rc in (N.MOE_EINVAL, N.MOE_ESPACE) and not handle.value and N.last_error()


@pytest.mark.parametrize("bad,groups,starts,prefixes", [
    ({}, -1, BASE, BASE), ({}, 1025, BASE, BASE), ({}, 3, None, BASE), ({}, 3, BASE, None), ({}, 3, BASE + 2, BASE),
    ({}, 3, BASE, BASE + 1), (dict(D=80), 3, BASE, BASE), (dict(lengths=None), 3, BASE, BASE), (dict(page=8), 3, BASE, BASE),
    (dict(workspace_bytes=128), 3, BASE, BASE), (dict(k_strides=(16384, 2048, 100)), 3, BASE, BASE),
])
def test_shared_refusals(bad, groups, starts, prefixes):
    handle = ctypes.c_void_p()
    rc = N.lib().gqa_shared_plan_create(ctypes.byref(handle), ctypes.byref(_paged(**bad)), groups, starts, prefixes)
    assert rc in (N.MOE_EINVAL, N.MOE_ESPACE) and not handle.value and N.last_error()


def test_attention_null_handles():
    lib, flags, size, handle = N.lib(), ctypes.c_uint32(), ctypes.c_size_t(), ctypes.c_void_p()
    for rc in (lib.gqa_shared_plan_run(None, None), lib.gqa_shared_plan_read_status(None, None, ctypes.byref(flags)),
               lib.gqa_paged_stored_plan_create(ctypes.byref(handle), ctypes.byref(_paged()), None),
               lib.gqa_shared_plan_create(None, ctypes.byref(_paged()), 0, BASE, BASE),
               lib.gqa_paged_stored_workspace_bytes(ctypes.byref(_paged()), 5, ctypes.byref(size)),
               lib.gqa_shared_workspace_bytes(ctypes.byref(_paged()), -2, ctypes.byref(size)),
               lib.gqa_shared_workspace_bytes(ctypes.byref(_paged()), 1, None)):
        assert rc == N.MOE_EINVAL and N.last_error()
    lib.gqa_shared_plan_destroy(None)
    assert ctypes.sizeof(N.GqaPagedScales) == 8 + 16 + 32  # int32 (+pad) + 2 pointers + 4 int64


def test_attention_python_refusals():
    q, pages = torch.zeros(6, 4, 128, dtype=torch.bfloat16), torch.zeros(9, 2, 16, 128, dtype=torch.bfloat16)
    tables, lengths = torch.zeros(6, 3, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    starts, prefixes = torch.tensor([0, 2, 6], dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad in [(starts.long(), prefixes), (starts, prefixes.long()), (starts, None)]:
        with pytest.raises(TypeError):
            prepare_shared_gqa(q, pages, pages, tables, lengths, *bad)
    eight = torch.zeros(9, 2, 16, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(TypeError):  # the shared form has 16-bit pages
        prepare_shared_gqa(q, eight, eight, tables, lengths, starts, prefixes)
    for bad in [(starts[:0], prefixes), (starts[None], prefixes), (starts, prefixes[:1]), (starts[:2], prefixes),
                (None, prefixes), (starts, prefixes)]:  # the last: not on a GPU
        with pytest.raises(ValueError):
            prepare_shared_gqa(q, pages, pages, tables, lengths, *bad)
    with pytest.raises(ValueError, match="scale"):
        prepare_shared_gqa(q, pages, pages, tables, lengths, starts, prefixes, scale=-1.0)
    with pytest.raises(ValueError, match="share storage"):
        prepare_shared_gqa(q, pages, pages, tables, lengths, starts, prefixes, out=q)
    scales = torch.zeros(9, 2, 4, 16, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(TypeError):
        prepare_paged_gqa(q, pages, pages, tables, lengths, k_scales=scales, v_scales=scales)
    with pytest.raises(TypeError):
        prepare_paged_gqa(q, eight, eight, tables, lengths, k_scales=scales)
    with pytest.raises(ValueError):  # not on a GPU
        prepare_paged_gqa(q, eight, eight, tables, lengths, k_scales=scales, v_scales=scales)


WITHOUT = r"""
import sys
import torch
for name in sys.argv[1].split(","):
    delattr(torch, name)
from llm_gpu_kernels_amd import PagedKVCache, prepare_paged_gqa, prepare_moe
sizes = dict(sequences=4, max_pages=8, max_tokens=64)
for storage, needs in ((None, ""), ("mxfp8", "float8_e4m3fn,float8_e8m0fnu"), ("mxfp4", "float4_e2m1fn_x2,float8_e8m0fnu")):
    try:
        PagedKVCache(10, 16, 2, 64, storage=storage, device="cpu", **sizes)
    except Exception as e:
        print(type(e).__name__, e, flush=True)
    gone = [n for n in needs.split(",") if n in sys.argv[1].split(",")]
    if not gone:
        continue
    try:
        q, t = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 16, 64, dtype=torch.uint8)
        prepare_paged_gqa(q, t, t, q, q, k_scales=t, v_scales=t)
    except TypeError as e:
        print("attention", e, flush=True)
"""


@pytest.mark.parametrize("gone", ["float4_e2m1fn_x2", "float8_e8m0fnu", "float4_e2m1fn_x2,float8_e8m0fnu,float8_e4m3fn"])
def test_a_torch_without_the_types_of_a_storage(gone):
    """The package is imported, and everything else of it works; a storage whose types are
    missing is refused by name."""
    done = subprocess.run([sys.executable, "-c", WITHOUT, gone], capture_output=True, text=True, cwd=ROOT)
    assert done.returncode == 0, done.stderr
    lines = done.stdout.splitlines()
    caches = [x for x in lines if not x.startswith("attention")]
    assert len(caches) == 3 and caches[0] == "ValueError device must be a GPU device"
    for line, needs in zip(caches[1:], ({"float8_e4m3fn", "float8_e8m0fnu"}, {"float4_e2m1fn_x2", "float8_e8m0fnu"})):
        missing = needs & set(gone.split(","))
        assert line.startswith("RuntimeError" if missing else "ValueError device") and all(f"torch.{n}" in line for n in missing)
    assert any(x.startswith("attention") for x in lines)
