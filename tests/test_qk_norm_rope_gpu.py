"""Norms and rotation of queries and keys against the same in 64 bits (MI355X only).

Tolerances.  Before the last rounding a value comes from fp32 operations: the sum of up
to 128 squares and its root (at most 66 roundings of 2^-24 relative, since the root
halves them), four more for the reciprocal root, the scaling and the weight, and in the
rotation two products, one sum and sines and cosines that are off by 2^-22 (half a turn
is rounded to fp32, then two units in the last place): less than 2^-17 of |y_l| + |y_h|.
The rounding to the type is off by half a step, eps / 2 of the value (fp16 below 2^-14:
2^-25), e4m3 by 2^-4 of the value or 2^-10 of the scale, e2m1 by 2^-2 of the value or a
quarter of the scale."""
import random

import pytest
import torch

from llm_gpu_kernels_amd import PagedKVCache, prepare_qk_norm_rope
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]
FP32 = 2.0 ** -17


def _inputs(n, hq, hkv, d, r, dtype, device, fused=True, norm=True, far=2 ** 17, weight_type=None, seed=0):
    g = torch.Generator().manual_seed(seed + n + r)
    rows = torch.randn(n, hq + 2 * hkv, d, generator=g) * torch.exp(torch.randn(n, hq + 2 * hkv, 1, generator=g))
    rows = rows.to(dtype).to(device)
    q, k, v = rows.split([hq, hkv, hkv], dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    positions = torch.randint(0, far, (n,), generator=g, dtype=torch.int32).to(device)
    inv_freq = torch.tensor([1e6 ** (-2 * i / r) for i in range(r // 2)], dtype=torch.float32, device=device)
    weights = [(1 + 0.3 * torch.randn(d, generator=g)).to(weight_type or dtype).to(device) if norm else None
               for _ in range(2)]
    return q, k, v, positions, inv_freq, weights


def _near(out, x, positions, inv_freq, weight, eps=1e-6, interleaved=False, step=None):
    """out against the 64-bit rows; step(ref): what the last rounding may do."""
    ref, size = S.norm_rope(x.cpu(), positions.cpu(), inv_freq.cpu(), None if weight is None else weight.cpu(), eps,
                            interleaved)
    tol = size * FP32
    if step is None:
        u = torch.finfo(out.dtype).eps / 2
        tol = tol * (1 + u) + u * ref.abs() + (2.0 ** -25 if out.dtype == torch.float16 else 0.0)
    else:
        tol = tol + step(ref)
    off = (out.double().cpu() - ref).abs()
    assert torch.isfinite(out).all()
    worst = (off / tol.clamp(min=1e-30)).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hkv,d,r", [(32, 8, 128, 128), (4, 4, 128, 64), (8, 1, 128, 2), (14, 2, 64, 64), (6, 6, 64, 32),
                                        (12, 4, 64, 26), (5, 1, 128, 90), (1, 1, 64, 16), (3, 3, 128, 112)])
def test_rows(hq, hkv, d, r, interleaved, dtype, gpu_device):
    q, k, _, positions, inv_freq, w = _inputs(37, hq, hkv, d, r, dtype, gpu_device, fused=hq != 4)
    plan = prepare_qk_norm_rope(q, k, positions, inv_freq, *w, interleaved=interleaved)
    q_out, k_out = plan.run()
    assert q_out.shape == q.shape and k_out.shape == k.shape and q_out.is_contiguous()
    _near(q_out, q, positions, inv_freq, w[0], interleaved=interleaved)
    _near(k_out, k, positions, inv_freq, w[1], interleaved=interleaved)


@pytest.mark.parametrize("n", [1, 2, 17, 300, 2000])
@pytest.mark.parametrize("norm", ["both", "q", "k", "none", "fp32"])
def test_weights_and_lengths(norm, n, gpu_device):
    q, k, _, positions, inv_freq, (a, b) = _inputs(n, 8, 2, 128, 128, torch.bfloat16, gpu_device,
                                                   weight_type=torch.float32 if norm == "fp32" else None)
    a, b = a if norm in ("both", "q", "fp32") else None, b if norm in ("both", "k", "fp32") else None
    q_out, k_out = prepare_qk_norm_rope(q, k, positions, inv_freq, a, b, eps=1e-3).run()
    _near(q_out, q, positions, inv_freq, a, 1e-3)
    _near(k_out, k, positions, inv_freq, b, 1e-3)


@pytest.mark.parametrize("far", [2 ** 24 + 5, 2 ** 31 - 1])
def test_far_positions(far, gpu_device):
    """The angle keeps its fraction of a turn: fp32 products would have none left."""
    q, k, _, positions, inv_freq, w = _inputs(40, 4, 2, 128, 128, torch.float16, gpu_device, far=far)
    positions[0], positions[1], positions[2] = far, 0, -far
    q_out, _ = prepare_qk_norm_rope(q, k, positions, inv_freq, *w).run()
    _near(q_out, q, positions, inv_freq, w[0])


def test_extreme_rows(gpu_device):
    """Rows of zeros stay zeros; tiny ones are held up by eps; a NaN or an infinity
    stays in its head."""
    q, k, _, positions, inv_freq, w = _inputs(9, 4, 2, 64, 64, torch.bfloat16, gpu_device, fused=False)
    q[0] = 0
    q[1] = 2.0 ** -120
    clean = prepare_qk_norm_rope(q, k, positions, inv_freq, *w)
    assert (clean.q_out[0] == 0).all()
    _near(clean.q_out, q, positions, inv_freq, w[0])
    before = clean.q_out.clone()
    q[2, 1, 7], q[3, 0, 0] = float("nan"), float("inf")
    out, _ = clean.run()
    # An infinite mean: finite elements over it are 0, the infinity over it is NaN, and so
    # is its pair.
    pair = torch.zeros(64, dtype=torch.bool, device=gpu_device)
    pair[0] = pair[32] = True
    assert torch.isnan(out[2, 1]).all() and torch.equal(torch.isnan(out[3, 0]), pair) and (out[3, 0][~pair] == 0).all()
    before[2, 1] = before[3, 0] = out[2, 1] = out[3, 0] = 0
    assert torch.equal(out, before)


def _cached(device, dtype, storage, n, hkv, d, page=16, layers=2):
    c = PagedKVCache(-(-n // page) + 2, page, hkv, d, sequences=1, max_pages=-(-n // page) + 2, max_tokens=n + 3,
                     layers=layers, dtype=dtype, storage=storage, device=device)
    slots = random.Random(n).sample(range(c.pages * page), n)
    if n > 2:
        slots[1], slots[2] = -1, c.pages * page  # nowhere, and outside the cache
    c.slots[:n] = torch.tensor(slots, device=device)
    return c, slots


def _held(c, t, scales, slots, layer):
    """Rows of the cache [n, heads, d] in 64 bits, and their scales."""
    s = torch.tensor(slots)
    p, r = s // c.page_size, s % c.page_size
    if c.storage is None:
        return t[layer].cpu()[p, :, r], None
    b = scales.view(torch.uint8)[layer].cpu()[p, :, :, r]
    codes = S.mx_unpack(t.view(torch.uint8)[layer].cpu()[p, :, r], c.storage)
    return S.mx_values(codes, b, c.storage), b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("storage", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hkv,d,r", [(1, 8, 2, 128, 128), (40, 4, 4, 64, 64), (700, 6, 2, 128, 32), (33, 3, 1, 64, 38),
                                          (600, 32, 8, 128, 128)])
def test_into_a_cache(n, hq, hkv, d, r, interleaved, storage, dtype, gpu_device):
    q, k, v, positions, inv_freq, w = _inputs(n, hq, hkv, d, r, dtype, gpu_device)
    c, slots = _cached(gpu_device, dtype, storage, n, hkv, d)
    rows = prepare_qk_norm_rope(q, k, positions, inv_freq, *w, interleaved=interleaved)
    plan = prepare_qk_norm_rope(q, k, positions, inv_freq, *w, interleaved=interleaved, v=v, cache=c, layer=1)
    q_out, k_out = plan.run()
    assert k_out is None and torch.equal(q_out, rows.q_out)
    kept = torch.tensor([0 <= s < c.pages * c.page_size for s in slots])
    slots = [s for s in slots if 0 <= s < c.pages * c.page_size]
    keys, ks = _held(c, c.k, c.k_scales, slots, 1)
    values, vs = _held(c, c.v, c.v_scales, slots, 1)
    if storage is None:
        assert torch.equal(keys, rows.k_out.cpu()[kept]) and torch.equal(values, v.cpu()[kept])
    else:
        codes, b = S.mx_quantise(v.cpu()[kept], storage, dtype)
        assert torch.equal(b, vs) and torch.equal(values, S.mx_values(codes, b, storage))
        scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), ks.long() - 127).repeat_interleave(32, -1)
        relative, absolute = (2.0 ** -4, 2.0 ** -10) if storage == "mxfp8" else (2.0 ** -2, 0.25)
        _near(keys, k.cpu()[kept], positions.cpu()[kept], inv_freq, w[1], interleaved=interleaved,
              step=lambda ref: torch.maximum(relative * ref.abs(), absolute * scale))
        # No scale is larger than the keys need: half of it would not do, or is too small already.
        ref, size = S.norm_rope(k.cpu()[kept], positions.cpu()[kept], inv_freq.cpu(), w[1].cpu(), interleaved=interleaved)
        top = (ref.abs() + size * FP32).unflatten(-1, (-1, 32)).amax(-1)
        half = torch.pow(torch.tensor(2.0, dtype=torch.float64), ks.long() - 128)
        assert (top > (448.0 if storage == "mxfp8" else 6.0) * half).all()
    # Nothing else was written, no other layer either.
    assert (c.k[0].view(torch.uint8) == 0).all() and (c.v[0].view(torch.uint8) == 0).all()
    free = torch.ones(c.pages * c.page_size, dtype=torch.bool)
    free[torch.tensor(slots)] = False
    for t in (c.k, c.v):
        flat = t.view(torch.uint8)[1].cpu().transpose(1, 2).reshape(c.pages * c.page_size, -1)
        assert (flat[free] == 0).all()


def test_keys_out_beside_a_cache(gpu_device):
    q, k, v, positions, inv_freq, w = _inputs(20, 8, 2, 128, 128, torch.bfloat16, gpu_device)
    c, _ = _cached(gpu_device, torch.bfloat16, "mxfp8", 20, 2, 128)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=gpu_device)
    plan = prepare_qk_norm_rope(q, k, positions, inv_freq, *w, k_out=k_out, v=v, cache=c)
    assert plan.run()[1] is k_out
    _near(k_out, k, positions, inv_freq, w[1])


def test_values_that_are_nan_keep_their_bits(gpu_device):
    q, k, v, positions, inv_freq, w = _inputs(5, 2, 2, 64, 64, torch.float16, gpu_device, fused=False)
    v.view(torch.int16)[2, 1, 3] = 0x7dab
    c, slots = _cached(gpu_device, torch.float16, None, 5, 2, 64)
    c.slots[:5] = torch.arange(5, device=gpu_device)
    prepare_qk_norm_rope(q, k, positions, inv_freq, *w, v=v, cache=c)
    assert torch.equal(c.v[0, 0, :, :5].transpose(0, 1).contiguous().view(torch.int16), v.view(torch.int16))


def test_no_tokens(gpu_device):
    q, k, v, positions, inv_freq, w = _inputs(4, 8, 2, 128, 128, torch.bfloat16, gpu_device)
    q_out, k_out = prepare_qk_norm_rope(q[:0], k[:0], positions[:0], inv_freq, *w).run()
    assert q_out.shape == (0, 8, 128) and k_out.shape == (0, 2, 128)
    c, _ = _cached(gpu_device, torch.bfloat16, None, 4, 2, 128)
    assert prepare_qk_norm_rope(q[:0], k[:0], positions[:0], inv_freq, v=v[:0], cache=c).run()[1] is None


def test_captured(gpu_device):
    """Replays with other values, positions and slots, on a stream of their own."""
    q, k, v, positions, inv_freq, w = _inputs(30, 8, 2, 128, 64, torch.bfloat16, gpu_device, fused=False)
    c, _ = _cached(gpu_device, torch.bfloat16, None, 30, 2, 128)
    plan = prepare_qk_norm_rope(q, k, positions, inv_freq, *w, v=v, cache=c)
    stream, graph = torch.cuda.Stream(gpu_device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        plan.run()
    for seed in range(3):
        other = _inputs(30, 8, 2, 128, 64, torch.bfloat16, gpu_device, fused=False, seed=100 + seed)
        for t, new in zip((q, k, v, positions), other[:4]):
            t.copy_(new)
        slots = random.Random(seed).sample(range(c.pages * 16), 30)
        c.slots[:30] = torch.tensor(slots, device=gpu_device)
        plan.q_out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _near(plan.q_out, q, positions, inv_freq, w[0])
        keys, _ = _held(c, c.k, None, slots, 0)
        _near(keys, k, positions, inv_freq, w[1])
        assert torch.equal(_held(c, c.v, None, slots, 0)[0], v.cpu())


def test_refusals_with_a_cache(gpu_device):
    q, k, v, positions, inv_freq, w = _inputs(20, 8, 2, 128, 128, torch.bfloat16, gpu_device, fused=False)
    c, _ = _cached(gpu_device, torch.bfloat16, "mxfp8", 17, 2, 128)
    small, _ = _cached(gpu_device, torch.bfloat16, None, 16, 2, 128)
    other, _ = _cached(gpu_device, torch.float16, None, 20, 2, 128)
    heads, _ = _cached(gpu_device, torch.bfloat16, None, 20, 4, 128)
    prepare_qk_norm_rope(q, k, positions, inv_freq, v=v, cache=c)
    for kw in (dict(v=v), dict(cache=c), dict(v=v[:5], cache=c), dict(v=v, cache=small), dict(v=v, cache=other),
               dict(v=v, cache=heads), dict(v=v, cache=c, layer=2), dict(v=v, cache=c, layer=-1), dict(q_out=q),
               dict(v=v, cache=c, k_out=v)):
        with pytest.raises(ValueError):
            prepare_qk_norm_rope(q, k, positions, inv_freq, **kw)
    flat = torch.empty(20 * 10 * 128, dtype=torch.bfloat16, device=gpu_device)
    q_out, k_out = flat[:20 * 8 * 128].view(q.shape), flat[20 * 8 * 128:].view(k.shape)
    prepare_qk_norm_rope(q, k, positions, inv_freq, q_out=q_out, k_out=k_out)
    with pytest.raises(ValueError, match="overlap"):
        prepare_qk_norm_rope(q, k, positions, inv_freq, q_out=q_out, k_out=flat[128:128 + k.numel()].view(k.shape))


@pytest.mark.parametrize("storage", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("down", [20, 24])
def test_small_fp16_keys_into_a_cache(down, interleaved, storage, gpu_device):
    """Keys quantised from fp32 below what fp16 holds: as near as the others in the cache, and
    read back to the nearest fp16 number.  Elements of four bits lie between fp16's numbers only
    where the largest of 32 is at most 6 * 2^-24 = 0.375 * 2^-20, so not among normed keys
    times 2^-20 and more."""
    n, hkv, d = 90, 2, 64
    q, k, v, positions, inv_freq, _ = _inputs(n, 4, hkv, d, d, torch.float16, gpu_device, fused=False)
    g = torch.Generator().manual_seed(8)
    weight = 2.0 ** -down * (1 + torch.rand(d, generator=g))
    c, slots = _cached(gpu_device, torch.float16, storage, n, hkv, d)
    slots = list(range(n))
    c.slots[:n] = torch.arange(n, device=gpu_device)
    prepare_qk_norm_rope(q, k, positions, inv_freq, None, weight.to(gpu_device), interleaved=interleaved, v=v, cache=c, layer=1)
    keys, b = _held(c, c.k, c.k_scales, slots, 1)
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), b.long() - 127).repeat_interleave(32, -1)
    relative, absolute = (2.0 ** -4, 2.0 ** -10) if storage == "mxfp8" else (2.0 ** -2, 0.25)
    _near(keys, k, positions, inv_freq, weight, interleaved=interleaved,
          step=lambda ref: torch.maximum(relative * ref.abs(), absolute * scale))
    off = (keys.half().double() - keys).abs()
    top = keys.abs().unflatten(-1, (-1, 32)).amax(-1)
    small = top <= (448 * 2.0 ** -16 if storage == "mxfp8" else 6 * 2.0 ** -24)  # what the type may not hold
    assert small.any() == (storage == "mxfp8" or down == 24) and (off <= 2.0 ** -25).all()
    assert (off > 0).any() == small.any() and (off.unflatten(-1, (-1, 32)).amax(-1)[~small] == 0).all()
    c.tables[0, :c.pages], c.lengths[0] = torch.arange(c.pages, dtype=torch.int32, device=gpu_device), n
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    at = [torch.tensor(x, dtype=torch.int32, device=gpu_device) for x in ([0], [0, n])]
    c.gather(1, *at, ko, vo)
    assert torch.equal(ko.cpu(), keys.half())


@pytest.mark.parametrize("storage", ["rows", None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("n,hq,hkv,d", [(2500, 32, 8, 128), (3000, 32, 8, 128), (5200, 8, 2, 128), (5200, 12, 4, 64),
                                        (8191, 24, 4, 128), (5121, 5, 5, 64), (900, 130, 2, 64), (6000, 2, 1, 128)])
def test_a_chunk_of_tokens(n, hq, hkv, d, storage, gpu_device):
    """As many tokens as have their heads in one wave, or shared out over a few: every row the
    same bits as in calls of 200 tokens, which are shared out more, and those as near as any."""
    interleaved = hq % 8 == 0
    q, k, v, positions, inv_freq, w = _inputs(n, hq, hkv, d, d, torch.bfloat16, gpu_device)
    at = list(range(0, n, 200))
    few = [prepare_qk_norm_rope(q[a:a + 200], k[a:a + 200], positions[a:a + 200], inv_freq, *w, interleaved=interleaved) for a in at]
    want_q, want_k = torch.cat([x.q_out for x in few]), torch.cat([x.k_out for x in few])
    for i in (0, len(few) - 1):
        a = slice(at[i], at[i] + 200)
        _near(few[i].q_out, q[a], positions[a], inv_freq, w[0], interleaved=interleaved)
        _near(few[i].k_out, k[a], positions[a], inv_freq, w[1], interleaved=interleaved)
    if storage == "rows":
        plan = prepare_qk_norm_rope(q, k, positions, inv_freq, *w, interleaved=interleaved)
        assert torch.equal(plan.q_out, want_q) and torch.equal(plan.k_out, want_k)
        return
    c, slots = _cached(gpu_device, torch.bfloat16, storage, n, hkv, d)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=gpu_device)
    plan = prepare_qk_norm_rope(q, k, positions, inv_freq, *w, interleaved=interleaved, k_out=k_out, v=v, cache=c, layer=1)
    assert torch.equal(plan.q_out, want_q) and torch.equal(k_out, want_k)
    planes = [t.view(torch.uint8).clone() for t in (c.k, c.v, c.k_scales, c.v_scales) if t is not None]
    for t in (c.k, c.v, c.k_scales, c.v_scales):
        if t is not None:
            t.view(torch.uint8).zero_()
    every = c.slots.clone()
    for a in at:  # the cache by calls of few tokens
        m = min(200, n - a)
        c.slots[:m] = every[a:a + m]
        prepare_qk_norm_rope(q[a:a + m], k[a:a + m], positions[a:a + m], inv_freq, *w, interleaved=interleaved, v=v[a:a + m], cache=c,
                             layer=1)
    for t, x in zip((c.k, c.v, c.k_scales, c.v_scales), planes):
        assert torch.equal(t.view(torch.uint8), x)


@pytest.mark.parametrize("storage", ["mxfp8", "mxfp4"])
def test_outputs_in_the_cache_are_refused(storage, gpu_device):
    """Its scales are written as its elements are."""
    q, k, v, positions, inv_freq, w = _inputs(20, 8, 2, 128, 128, torch.bfloat16, gpu_device, fused=False)
    c = PagedKVCache(600, 16, 2, 128, sequences=1, max_pages=2, max_tokens=20, storage=storage, device=gpu_device)
    for held in (c.k, c.v, c.k_scales, c.v_scales):
        flat = held.view(torch.uint8).flatten().view(torch.bfloat16)
        for kw in (dict(q_out=flat[:q.numel()].view(q.shape)), dict(k_out=flat[-k.numel():].view(k.shape))):
            with pytest.raises(ValueError, match="share storage"):
                prepare_qk_norm_rope(q, k, positions, inv_freq, *w, v=v, cache=c, **kw)
        assert (held.view(torch.uint8) == 0).all()


def test_as_many_tokens_as_allowed(gpu_device):
    """2^24 tokens, the same 1024 over and over: every time the same bits."""
    q, k, _, positions, inv_freq, w = _inputs(1024, 2, 1, 64, 64, torch.bfloat16, gpu_device)
    few = prepare_qk_norm_rope(q, k, positions, inv_freq, *w)
    times = 2 ** 14
    plan = prepare_qk_norm_rope(q.repeat(times, 1, 1), k.repeat(times, 1, 1), positions.repeat(times), inv_freq, *w)
    for out, one in ((plan.q_out, few.q_out), (plan.k_out, few.k_out)):
        assert (out.view(times, *one.shape).view(torch.int16) == one.view(torch.int16)).all()
