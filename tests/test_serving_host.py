"""Packed and paged attention and the paged cache without a GPU: refusals of the
C ABI and of the Python layer, and the oracle's own invariants."""
import ctypes
import random

import pytest
import torch

from llm_gpu_kernels_amd import PagedKVCache, _native as N, prepare_packed_gqa, prepare_paged_gqa
from oracle import serving_oracle as S

BASE = 1 << 20  # an address that is only looked at by the validation


def test_struct_sizes_match_header():
    # 6 int32 + 5 pointers + 3 int64 + float (+pad) + pointer + size_t.
    assert ctypes.sizeof(N.GqaPackedDesc) == 24 + 40 + 24 + 8 + 16
    # 8 int32 + 6 pointers + 8 int64 + float (+pad) + pointer + size_t.
    assert ctypes.sizeof(N.GqaPagedDesc) == 32 + 48 + 64 + 8 + 16
    # 8 int32 + 9 pointers + size_t.
    assert ctypes.sizeof(N.KvCacheDesc) == 32 + 72 + 8


def _packed(**kw):
    d = N.GqaPackedDesc()
    d.N, d.S, d.Hq, d.Hkv, d.D, d.dtype = 100, 3, 32, 8, 128, N.GQA_BF16
    d.q = d.k = d.v = d.out = d.starts = d.workspace = BASE
    d.q_stride, d.k_stride, d.v_stride = 4096, 1024, 1024
    d.workspace_bytes = 1 << 30
    for name, value in kw.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("bad", [
    dict(D=96), dict(D=256), dict(Hq=31), dict(Hkv=0), dict(Hq=0), dict(Hq=65, Hkv=1), dict(dtype=2), dict(N=-1),
    dict(N=1 << 29), dict(N=1 << 24), dict(S=1 << 20, N=1 << 22, Hq=32, Hkv=32), dict(S=-1), dict(S=(1 << 20) + 1), dict(q=None), dict(k=BASE + 8), dict(out=None), dict(starts=None),
    dict(starts=BASE + 2), dict(q_stride=4088), dict(k_stride=1028), dict(v_stride=0), dict(k_stride=(1 << 25) + 8),
    dict(workspace=None), dict(workspace_bytes=0),
])
def test_packed_refusals(bad):
    handle = ctypes.c_void_p()
    rc = N.lib().gqa_packed_plan_create(ctypes.byref(handle), ctypes.byref(_packed(**bad)))
    assert rc in (N.MOE_EINVAL, N.MOE_ESPACE) and not handle.value and N.last_error()


def _paged(**kw):
    d = N.GqaPagedDesc()
    d.B, d.Hq, d.Hkv, d.D, d.P, d.page, d.M, d.dtype = 5, 32, 8, 128, 100, 16, 20, N.GQA_BF16
    d.q = d.k = d.v = d.out = d.tables = d.lengths = d.workspace = BASE
    d.q_stride, d.table_stride = 4096, 20
    for st in (d.k_strides, d.v_strides):
        st[0], st[1], st[2] = 16 * 8 * 128, 16 * 128, 128
    d.workspace_bytes = 1 << 30
    for name, value in kw.items():
        if name in ("k_strides", "v_strides"):
            value = (ctypes.c_int64 * 3)(*value)
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("bad", [
    dict(D=80), dict(Hq=12), dict(Hq=520, Hkv=8), dict(dtype=-1), dict(B=-1), dict(B=(1 << 16) + 1), dict(page=0),
    dict(page=8), dict(page=24), dict(page=2048), dict(P=0), dict(M=0), dict(M=1 << 27), dict(M=1 << 22), dict(B=1 << 16, Hq=1024, Hkv=1024, M=1), dict(q=None), dict(k=BASE + 4),
    dict(v=None), dict(tables=None), dict(lengths=BASE + 1), dict(table_stride=19), dict(q_stride=4092),
    dict(k_strides=(16384, 2048, 120)), dict(k_strides=(0, 2048, 128)), dict(v_strides=(16384, 2044, 128)),
    dict(v_strides=(16384, 2048, (1 << 25) + 8)), dict(workspace=None), dict(workspace_bytes=0),
])
def test_paged_refusals(bad):
    handle = ctypes.c_void_p()
    rc = N.lib().gqa_paged_plan_create(ctypes.byref(handle), ctypes.byref(_paged(**bad)))
    assert rc in (N.MOE_EINVAL, N.MOE_ESPACE) and not handle.value and N.last_error()


def _cache(**kw):
    d = N.KvCacheDesc()
    d.pages, d.page_size, d.kv_heads, d.head_dim, d.layers = 100, 16, 8, 128, 2
    d.sequences, d.max_pages, d.max_tokens = 4, 10, 64
    for name in ("k", "v", "tables", "lengths", "refs", "starts", "slots", "status", "workspace"):
        setattr(d, name, BASE)
    d.workspace_bytes = 1 << 30
    for name, value in kw.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("bad", [
    dict(pages=0), dict(pages=N.KV_MAX_PAGES + 1), dict(page_size=0), dict(page_size=20), dict(page_size=2048),
    dict(head_dim=96), dict(kv_heads=0), dict(layers=0), dict(sequences=0), dict(sequences=N.KV_MAX_SEQUENCES + 1),
    dict(max_pages=0), dict(max_pages=1 << 27), dict(max_tokens=0), dict(max_tokens=N.KV_MAX_TOKENS + 1), dict(k=None),
    dict(v=BASE + 8), dict(tables=None), dict(refs=BASE + 4), dict(slots=BASE + 4), dict(status=None),
    dict(workspace=None), dict(workspace_bytes=16),
])
def test_cache_refusals(bad):
    handle = ctypes.c_void_p()
    rc = N.lib().kv_cache_create(ctypes.byref(handle), ctypes.byref(_cache(**bad)))
    assert rc in (N.MOE_EINVAL, N.MOE_ESPACE) and not handle.value and N.last_error()


def test_null_handles():
    lib, flags = N.lib(), ctypes.c_uint32()
    for rc in (lib.gqa_packed_plan_run(None, None), lib.gqa_paged_plan_run(None, None),
               lib.gqa_packed_plan_read_status(None, None, ctypes.byref(flags)), lib.kv_cache_compact(None, None),
               lib.kv_cache_reserve(None, BASE, 0, None), lib.kv_cache_fork(None, BASE, BASE, 1, None),
               lib.kv_cache_free(None, BASE, 1, None), lib.kv_cache_append(None, 0, BASE, BASE, 1024, 1024, 1, None),
               lib.kv_cache_read_status(None, None, ctypes.byref(flags)),
               lib.gqa_packed_workspace_bytes(None, None), lib.kv_cache_workspace_bytes(ctypes.byref(_cache()), None)):
        assert rc == N.MOE_EINVAL and N.last_error()
    lib.gqa_packed_plan_destroy(None)
    lib.gqa_paged_plan_destroy(None)
    lib.kv_cache_destroy(None)


def _rows(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def test_python_refusals():
    q, k, starts = _rows(6, 4, 128), _rows(6, 2, 128), torch.tensor([0, 6], dtype=torch.int32)
    with pytest.raises(TypeError):
        prepare_packed_gqa(q.float(), k, k, starts)
    with pytest.raises(TypeError):
        prepare_packed_gqa(q, k, k, starts.long())
    for bad in [(q[:, :, :100], k, k, starts), (q, k[:5], k[:5], starts), (q, k, k.half(), starts),
                (q, k, _rows(6, 1, 128), starts), (q, k, k, starts[None]), (q, k, k, starts[:0]),
                (_rows(6, 128, 4).transpose(1, 2), k, k, starts), (_rows(6, 3, 128), k, k, starts), (q, k, k, starts)]:
        with pytest.raises(ValueError):  # the last: not on a GPU
            prepare_packed_gqa(*bad)
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-45, 1e-50, 2e38, 1e39):
        with pytest.raises(ValueError, match="scale"):
            prepare_packed_gqa(q, k, k, starts, scale=scale)
    with pytest.raises(ValueError, match="share storage"):
        prepare_packed_gqa(q, k, k, starts, out=q)
    meta = q.to("meta")
    many = torch.zeros(1, dtype=torch.int32, device="meta").expand(2 ** 32 + 2).clone()
    with pytest.raises(ValueError, match="S must be below"):
        prepare_packed_gqa(meta, k.to("meta"), k.to("meta"), many)
    pages, tables, lengths = _rows(9, 2, 16, 128), torch.zeros(6, 3, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    with pytest.raises(TypeError):
        prepare_paged_gqa(q, pages, pages, tables.long(), lengths)
    for bad in [(q, pages, pages[:8], tables, lengths), (q, pages, pages, tables[:5], lengths),
                (q, pages, pages, tables, lengths[:5]), (q, pages[0], pages[0], tables, lengths),
                (q, pages.half(), pages.half(), tables, lengths), (q, pages, pages, tables[0], lengths),
                (q, pages, pages, tables, lengths)]:
        with pytest.raises(ValueError):
            prepare_paged_gqa(*bad)
    huge = pages[:1].to("meta").expand(2 ** 31, 2, 16, 128)
    with pytest.raises(ValueError, match="P must be below"):
        prepare_paged_gqa(meta, huge, huge, tables.to("meta"), lengths.to("meta"))
    good = dict(sequences=4, max_pages=8, max_tokens=64)
    with pytest.raises(TypeError):
        PagedKVCache(10, 16, 2, 64, dtype=torch.float32, **good)
    for args, kw in [((0, 16, 2, 64), {}), ((10, 8, 2, 64), {}), ((10, 16, 2, 96), {}), ((10, 16.0, 2, 64), {}),
                     ((10, 16, 2, 64), dict(sequences=2000)), ((10, 16, 2, 64), dict(device="cpu"))]:
        with pytest.raises(ValueError):
            PagedKVCache(*args, **{**good, **kw})


def test_oracle_invariants():
    """Random calls keep the oracle's holders, tables and lengths consistent, and
    a refused reserve changes nothing."""
    rng = random.Random(3)
    c = S.Cache(40, 16, 6, 12, 200)
    refused = 0
    for _ in range(400):
        what = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        if what == "reserve":
            before = (list(c.lengths), [list(t) for t in c.tables], list(c.refs))
            c.status = 0
            c.reserve([rng.choice([0, 0, 1, 5, 40]) for _ in range(6)])
            if c.status:
                refused += 1
                assert before == (c.lengths, c.tables, c.refs) and set(c.slots) == {-1}
        elif what == "fork":
            c.fork([rng.randrange(-1, 7) for _ in range(3)], [rng.randrange(-1, 7) for _ in range(3)])
        elif what == "free":
            c.free([rng.randrange(-1, 7) for _ in range(2)])
        else:
            c.compact()
            assert all(r > 0 for r in c.refs[:sum(x > 0 for x in c.refs)])
        c.check()
    assert 10 < refused < 200


def test_oracle_copy_on_write():
    """Three rows share a partly filled page: two that grow get copies, and when
    all three grow the last keeps it."""
    c = S.Cache(10, 16, 4, 4, 64)
    c.reserve([5, 0, 0, 0])
    c.fork([0, 0], [1, 2])
    assert c.refs[0] == 3
    c.reserve([1, 1, 1, 0], stride=1)
    assert c.moves == [(0, 1), (0, 2)] and c.tables[:3] == [[1], [2], [0]] and c.refs[:3] == [1, 1, 1]
    assert c.slots[:4] == [21, 37, 5, -1] and c.starts == [0, 1, 2, 3, 3]
    c.free([0, 2])
    c.compact()
    assert c.moves == [(2, 0)] and c.tables[1] == [0] and c.refs[0] == 1
