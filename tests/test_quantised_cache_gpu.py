"""The paged cache with microscaled storage, and rows of any cache read back:
elements and scales exactly (MI355X only)."""
import random

import pytest
import torch

from llm_gpu_kernels_amd import PagedKVCache, _native as N
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu

STORAGES = ["mxfp8", "mxfp4"]
TYPES = [torch.bfloat16, torch.float16]


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _cache(device, storage, dtype=torch.bfloat16, pages=12, page=16, heads=2, dim=64, sequences=4, max_pages=12,
           max_tokens=200, layers=2):
    c = PagedKVCache(pages, page, heads, dim, sequences=sequences, max_pages=max_pages, max_tokens=max_tokens, layers=layers,
                     dtype=dtype, storage=storage, device=device)
    for t in _planes(c):  # what a call leaves out keeps these
        t.view(torch.uint8).fill_(0x5a)
    return c


def _planes(c):
    return [t for t in (c.k, c.v, c.k_scales, c.v_scales) if t is not None]


def _bytes(t):
    return t.view(torch.uint8).cpu()


def _tokens(n, heads, dim, dtype, seed):
    """Blocks of every magnitude that the type has, zeros and signed zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=g, dtype=torch.float64)
    low, high = (-130, 127) if dtype == torch.bfloat16 else (-24, 15)
    e = torch.randint(low, high, (n, heads, dim // 32, 1), generator=g)
    e = torch.where(torch.rand(e.shape, generator=g) < 0.5, 0, e)
    x = x.unflatten(-1, (-1, 32)) * torch.pow(torch.tensor(2.0, dtype=torch.float64), e)
    x = torch.where(torch.rand(x.shape, generator=g) < 0.05, x * 2.0 ** -9, x)
    x = torch.where(torch.rand(x.shape, generator=g) < 0.05, -0.0, x).flatten(-2)
    limit = torch.finfo(dtype).max
    return x.clamp(-limit, limit).to(dtype)


def _write(held, scales, storage, dtype, layer, slots, rows, page):
    """An append, by the oracle, into copies of a cache's bytes."""
    codes, exponents = S.mx_quantise(rows, storage, dtype)
    codes = S.mx_pack(codes, storage)
    for i, slot in enumerate(slots):
        if slot >= 0:
            held[layer, slot // page, :, slot % page] = codes[i]
            scales[layer, slot // page, :, :, slot % page] = exponents[i]


def _check_append(c, slots, k, v, layer):
    page = c.page_size
    want = [_bytes(t) for t in _planes(c)]
    c.slots[:len(slots)] = torch.tensor(slots, device=c.device)
    c.append(layer, k, v)
    _write(want[0], want[2], c.storage, c.dtype, layer, slots, k.cpu(), page)
    _write(want[1], want[3], c.storage, c.dtype, layer, slots, v.cpu(), page)
    for got, expected in zip(_planes(c), want):
        assert torch.equal(_bytes(got), expected)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("heads,dim,page,n", [(2, 64, 16, 1), (1, 64, 16, 77), (8, 128, 48, 150), (3, 128, 16, 33),
                                              (5, 64, 80, 200)])
def test_append(heads, dim, page, n, storage, dtype, gpu_device):
    c = _cache(gpu_device, storage, dtype, pages=300 // page + 2, page=page, heads=heads, dim=dim)
    slots = random.Random(n).sample(range(c.pages * page), n)
    for i in range(0, n, 7):
        slots[i] = -1 if n > 1 else slots[i]
    rows = _tokens(n, 2 * heads, dim, dtype, n).to(gpu_device)  # k and v are views of one projection
    _check_append(c, slots, rows[:, :heads], rows[:, heads:], 1)


@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("dtype", TYPES)
def test_append_every_number(dtype, storage, gpu_device):
    """Every finite 16-bit pattern beside a neighbour that sets the scale: both as the
    largest of its block and as a smaller one."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(dtype)
    x = x[torch.isfinite(x)]
    n = len(x) // 64
    x = x[:n * 64]
    alone = torch.zeros(len(x), 32, dtype=dtype)
    alone[:, 5] = x
    beside = x.view(-1, 32)[:, torch.randperm(32, generator=torch.Generator().manual_seed(1))]
    rows = torch.cat([alone, beside]).view(-1, 1, 64)
    rows = torch.cat([rows, rows[:-len(rows) % 64 or None]])[:len(rows) // 64 * 64]
    page = 1024
    c = _cache(gpu_device, storage, dtype, pages=len(rows) // page + 1, page=page, heads=1, dim=64, max_pages=64,
               max_tokens=len(rows), layers=1)
    rows = rows.to(gpu_device)
    _check_append(c, list(range(len(rows))), rows, rows.flip(0).contiguous(), 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("storage", STORAGES)
def test_not_finite(storage, dtype, gpu_device):
    """A block with an infinity or a NaN reads back as NaN, its neighbours do not."""
    c = _cache(gpu_device, storage, dtype)
    k, v = (_tokens(16, 2, 64, dtype, i).to(gpu_device) for i in (1, 2))
    k[3, 1, 40], v[5, 0, 3], v[5, 1, 63] = float("inf"), float("nan"), float("-inf")
    _check_append(c, list(range(16)), k, v, 0)
    c.tables[0, 0], c.lengths[0] = 0, 16
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    c.gather(0, _i32([0], gpu_device), _i32([0, 16], gpu_device), ko, vo)
    bad = torch.zeros_like(k, dtype=torch.bool)
    bad[3, 1, 32:] = True
    assert torch.equal(torch.isnan(ko), bad)
    bad.zero_()
    bad[5, 0, :32] = bad[5, 1, 32:] = True
    assert torch.equal(torch.isnan(vo), bad)
    c.check_inputs()


def _filled(c, seed):
    """Random elements and scales that stand for finite numbers, in every page."""
    g = torch.Generator().manual_seed(seed)
    for t in (c.k, c.v):
        if c.storage is None:
            t.copy_(torch.randn(t.shape, generator=g))
        else:
            b = torch.randint(0, 256, t.view(torch.uint8).shape, generator=g, dtype=torch.uint8)
            if c.storage == "mxfp8":
                b[(b & 127) == 127] = 3
            t.view(torch.uint8).copy_(b)
    for t in (c.k_scales, c.v_scales):
        if t is not None:
            # fp16: products of e4m3 elements below 2^-24 round, which the oracle does not follow.
            low, high = (10, 240) if c.dtype == torch.bfloat16 else (112, 127)
            t.view(torch.uint8).copy_(torch.randint(low, high, t.shape, generator=g, dtype=torch.uint8))


def _rows_of(c, t, scales, layer, row, n):
    """The first n tokens of a row [n, heads, dim] as the cache's tokens' type."""
    table = c.tables[row].tolist()
    places = [(table[j // c.page_size], j % c.page_size) for j in range(n)]
    p, r = torch.tensor([x for x, _ in places], dtype=torch.long), torch.tensor([x for _, x in places], dtype=torch.long)
    if c.storage is None:
        return t[layer].cpu()[p, :, r]
    values = S.mx_values(S.mx_unpack(_bytes(t)[layer][p, :, r], c.storage), _bytes(scales)[layer][p, :, :, r], c.storage)
    return values.to(c.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("storage", [None] + STORAGES)
@pytest.mark.parametrize("heads,dim,page", [(1, 64, 16), (8, 128, 48), (3, 128, 32)])
def test_gather(heads, dim, page, storage, dtype, gpu_device):
    c = _cache(gpu_device, storage, dtype, pages=40, page=page, heads=heads, dim=dim, sequences=6, max_pages=9)
    _filled(c, heads)
    lengths = [1, 0, 5 * page, 3 * page + 7, page + 1, page - 1]
    order = random.Random(page).sample(range(40), 40)
    for i, n in enumerate(lengths):
        used = -(-n // page)
        c.tables[i, :used] = _i32([order.pop() for _ in range(used)], gpu_device)
    c.lengths.copy_(_i32(lengths, gpu_device))
    rows = [3, 0, -1, 3, 2, 1]                     # one twice, one negative, an empty one
    counts = [3 * page + 7, 4, 5, 20, 5 * page, 3]  # longer than the row, none of it, part of it
    starts = [2]
    for n in counts:
        starts.append(starts[-1] + n)
    n = starts[-1] + 3
    fused = torch.full((n, 2 * heads, dim), 7.0, dtype=dtype, device=gpu_device)
    k, v = fused[:, :heads], fused[:, heads:]
    want_k, want_v = k.cpu().clone(), v.cpu().clone()
    for row, at, count in zip(rows, starts, counts):
        m = min(count, lengths[row]) if row >= 0 else 0
        want_k[at:at + m] = _rows_of(c, c.k, c.k_scales, 1, row, m)
        want_v[at:at + m] = _rows_of(c, c.v, c.v_scales, 1, row, m)
    c.gather(1, _i32(rows, gpu_device), _i32(starts, gpu_device), k, v)
    assert torch.equal(k.cpu().view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(v.cpu().view(torch.int16), want_v.view(torch.int16))
    c.check_inputs()


def test_gather_nothing(gpu_device):
    c = _cache(gpu_device, "mxfp8")
    k = torch.full((5, 2, 64), 3.0, dtype=torch.bfloat16, device=gpu_device)
    v = k.clone()
    none = _i32([], gpu_device)
    c.gather(0, none, _i32([0], gpu_device), k, v)
    c.gather(0, _i32([0], gpu_device), _i32([0, 5], gpu_device), k, v)            # an empty row
    c.gather(0, _i32([0], gpu_device), _i32([0, 0], gpu_device), k[:0], v[:0])    # no tokens
    assert (k == 3).all() and (v == 3).all()
    c.check_inputs()


def test_gather_more_tokens_than_a_grid(gpu_device):
    """Refused before anything is launched."""
    c = _cache(gpu_device, "mxfp8")
    k = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=gpu_device)
    rows, starts, many = _i32([0], gpu_device), _i32([0, 1], gpu_device), N.KV_MAX_GATHER_TOKENS + 1
    with pytest.raises(ValueError, match="tokens"):
        c.gather(0, rows, starts, k.expand(many, 2, 64), k.expand(many, 2, 64))
    for tokens in (many, 2 ** 31 - 1, -1):
        assert N.lib().kv_cache_gather(c._cache, 0, rows.data_ptr(), starts.data_ptr(), 1, k.data_ptr(), k.data_ptr(), 128,
                                       128, tokens, None) == N.MOE_EINVAL
    c.check_inputs()


@pytest.mark.parametrize("what,status", [("page", N.KV_STATUS_BAD_STATE), ("length", N.KV_STATUS_BAD_STATE),
                                         ("row", N.KV_STATUS_BAD_ROW), ("starts", N.KV_STATUS_BAD_COUNT),
                                         ("behind", N.KV_STATUS_BAD_COUNT), ("negative", N.KV_STATUS_BAD_COUNT)])
def test_gather_bad_inputs(what, status, gpu_device):
    """Reported, and left out: the other row is read."""
    c = _cache(gpu_device, "mxfp4")
    _filled(c, 4)
    c.tables[:2, :2] = _i32([[4, 5], [6, 7]], gpu_device)
    c.lengths[:2] = 20
    rows, starts = [0, 1], [0, 20, 40]
    if what == "page":
        c.tables[1, 1] = 12
    elif what == "length":
        c.lengths[1] = 12 * 16 + 1
    elif what == "row":
        rows[1] = 4
    elif what == "starts":
        starts = [0, 20, 19]
    elif what == "behind":
        starts[2] = 2 ** 31 - 1
    else:
        starts = [-2 ** 31, 20, 40]
    k = torch.full((41, 2, 64), 3.0, dtype=torch.bfloat16, device=gpu_device)
    v = k.clone()
    c.gather(0, _i32(rows, gpu_device), _i32(starts, gpu_device), k, v)
    assert c.read_status() == status
    if what != "starts":
        first = _rows_of(c, c.k, c.k_scales, 0, 0, 20)
        assert torch.equal(k[:20].cpu(), first)
    assert (k[40:] == 3).all() and (v[40:] == 3).all()
    assert c.read_status() == 0


@pytest.mark.parametrize("storage", [None] + STORAGES)
def test_random_calls(storage, gpu_device):
    """Pages and their scales move together: copies of shared pages and compaction."""
    rng = random.Random(5)
    sequences, page, max_pages = 7, 16, 8
    c = _cache(gpu_device, storage, pages=40, page=page, heads=3, dim=128, sequences=sequences, max_pages=max_pages,
               layers=3)
    _filled(c, 9)
    ref = S.Cache(40, page, sequences, max_pages, 200)
    planes = [_bytes(t) for t in _planes(c)]
    moves = 0

    def call(name, *lists, **kw):
        nonlocal moves
        getattr(c, name)(*(_i32(x, gpu_device) for x in lists), **kw)
        getattr(ref, name)(*lists, **kw)
        for a, b in ref.moves:
            moves += 1
            for t in planes:
                t[:, b] = t[:, a]

    for _ in range(60):
        what = rng.choice(["reserve", "step", "fork", "fork", "free", "compact"])
        if what == "reserve":
            call("reserve", [rng.choice([0, 1, 9, 30]) for _ in range(sequences)])
        elif what == "step":
            call("reserve", [int(n > 0) for n in ref.lengths], stride=1)
        elif what == "fork":
            empty = [i for i, n in enumerate(ref.lengths) if n == 0]
            call("fork", [rng.randrange(sequences)], [rng.choice(empty) if empty else 0])
        elif what == "free":
            call("free", [rng.randrange(sequences)])
        else:
            call("compact")
        assert c.tables.tolist() == [t + [-1] * (max_pages - len(t)) for t in ref.tables]
        assert c.read_status() == ref.status
        ref.status = 0
        for got, want in zip(_planes(c), planes):
            assert torch.equal(_bytes(got), want)
    assert moves >= 5  # pages did move


@pytest.mark.parametrize("storage", STORAGES)
def test_captured_and_on_another_stream(storage, gpu_device):
    """append and gather in a graph, replayed with other values and slots."""
    c = _cache(gpu_device, storage, dim=128)
    c.tables[0, :2], c.lengths[0] = _i32([3, 8], gpu_device), 30
    k, v = (_tokens(30, 2, 128, torch.bfloat16, i).to(gpu_device) for i in (1, 2))
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    rows, starts = _i32([0], gpu_device), _i32([0, 30], gpu_device)
    slots = [3 * 16 + j if j < 16 else 8 * 16 + j - 16 for j in range(30)]
    c.slots[:30] = torch.tensor(slots, device=gpu_device)
    stream = torch.cuda.Stream(gpu_device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        c.append(0, k, v)
        c.gather(0, rows, starts, ko, vo)
        with torch.cuda.graph(graph, stream=stream):
            c.append(0, k, v)
            c.gather(0, rows, starts, ko, vo)
    for seed in range(4):
        k.copy_(_tokens(30, 2, 128, torch.bfloat16, 10 + seed))
        v.copy_(_tokens(30, 2, 128, torch.bfloat16, 20 + seed))
        ko.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for out, x in ((ko, k), (vo, v)):
            want = S.mx_values(*S.mx_quantise(x.cpu(), storage, x.dtype), storage).to(x.dtype)
            assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("storage", STORAGES)
def test_offsets_past_32_bits(storage, gpu_device):
    """The last pages of a cache whose elements fill more than 4 GiB."""
    page, pages = 1024, (1 << 17) if storage == "mxfp4" else (1 << 16)
    c = PagedKVCache(pages + 5, page, 1, 64 if storage == "mxfp8" else 128, sequences=2, max_pages=4, max_tokens=100,
                     storage=storage, device=gpu_device)
    assert c.k.numel() > 2 ** 32
    k, v = (_tokens(100, 1, c.head_dim, torch.bfloat16, i).to(gpu_device) for i in (1, 2))
    c.slots.copy_(torch.arange(100, device=gpu_device) + (pages + 4) * page + 500)
    c.append(0, k, v)
    c.tables[1, 0], c.lengths[1] = pages + 4, 600
    ko, vo = (torch.zeros(600, 1, c.head_dim, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    c.gather(0, _i32([1], gpu_device), _i32([0, 600], gpu_device), ko, vo)
    for out, x in ((ko, k), (vo, v)):
        want = S.mx_values(*S.mx_quantise(x.cpu(), storage, x.dtype), storage).to(x.dtype)
        assert torch.equal(out[500:].cpu(), want) and (out[:500] == 0).all()
    c.check_inputs()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("storage", STORAGES)
def test_gather_every_element_under_every_scale(storage, dtype, gpu_device):
    """In the tokens' type to nearest even: what that holds exactly, fp16 between its smallest
    numbers too, beyond its largest an infinity."""
    n = 1020
    c = _cache(gpu_device, storage, dtype, pages=2, page=1024, heads=1, sequences=1, max_pages=2, max_tokens=n, layers=1)
    codes = torch.arange(n * 64).view(n, 64) % (256 if storage == "mxfp8" else 16)
    scales = torch.arange(n) // 4  # 0 to 254
    held = S.mx_pack(codes.to(torch.uint8), storage)
    for t, s in ((c.k, c.k_scales), (c.v, c.v_scales)):
        t.view(torch.uint8)[0, 1, 0, :n] = held.to(gpu_device)
        s.view(torch.uint8)[0, 1, 0, :, :n] = scales.to(torch.uint8).expand(2, n).to(gpu_device)
    c.tables[0, 0], c.lengths[0] = 1, n
    k, v = (torch.zeros(n, 1, 64, dtype=dtype, device=gpu_device) for _ in range(2))
    c.gather(0, _i32([0], gpu_device), _i32([0, n], gpu_device), k, v)
    values = S.mx_values(codes, scales[:, None].expand(n, 2), storage)
    want = values.to(dtype)
    assert not torch.equal(want.double().nan_to_num(0), values.nan_to_num(0))  # some do not fit
    for out in (k, v):
        out = out[:, 0].cpu()
        assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("storage", STORAGES)
def test_small_fp16_tokens_read_back(storage, gpu_device):
    """What append writes of tokens down to fp16's smallest is read back without another rounding."""
    g = torch.Generator().manual_seed(6)
    c = _cache(gpu_device, storage, torch.float16)
    e = torch.randint(-24, -8, (2, 150, 2, 2, 1), generator=g).double()
    x = torch.randn(2, 150, 2, 2, 32, generator=g, dtype=torch.float64) * torch.pow(torch.tensor(2.0, dtype=torch.float64), e)
    k, v = x.flatten(-2).half().to(gpu_device)
    c.slots[:150] = torch.arange(150, device=gpu_device)
    c.append(0, k, v)
    c.tables[0, :10], c.lengths[0] = _i32(list(range(10)), gpu_device), 150
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    c.gather(0, _i32([0], gpu_device), _i32([0, 150], gpu_device), ko, vo)
    for out, x in ((ko, k), (vo, v)):
        assert torch.equal(out.double().cpu(), S.mx_values(*S.mx_quantise(x.cpu(), storage, x.dtype), storage))


@pytest.mark.parametrize("storage", [None] + STORAGES)
def test_gather_refuses_memory_that_is_read_or_written_twice(storage, gpu_device):
    """Before anything is launched; rows of one tensor between each other's are taken."""
    n, dim, heads = 40, 64, 1
    c = _cache(gpu_device, storage, heads=heads, dim=dim, layers=1)
    c.tables[0, :3], c.lengths[0] = _i32([3, 8, 5], gpu_device), n
    _filled(c, 5)
    rows, starts = _i32([0], gpu_device), _i32([0, n], gpu_device)
    want = [_rows_of(c, t, s, 0, 0, n) for t, s in ((c.k, c.k_scales), (c.v, c.v_scales))]
    before = [_bytes(t) for t in _planes(c)] + [t.cpu() for t in (c.tables, c.lengths, c.refs, c.slots, c.starts)]

    def new(*shape):
        return torch.zeros(*shape, dtype=c.dtype, device=gpu_device)

    def of(t):  # a tensor of the call's type at a tensor's memory, if it holds that many
        flat = t.reshape(-1).view(torch.uint8).view(c.dtype)
        return flat[:flat.numel() // dim * dim].view(-1, heads, dim)

    other, one, wide = new(n, heads, dim), new(2 * n, heads, dim), new(n + 1, heads, 2 * dim)
    taken = [(new(n, heads, dim), other), (wide[:n, :, dim:], wide[1:, :, :dim]), (one[:n], one[n:]), (one[n:], one[:n]), (one[0::2], one[1::2]), (one[1::2], one[0::2]),
             new(n, 2 * heads, dim).split(heads, 1), new(n, 3 * heads, dim)[:, 1:].split(heads, 1)]
    for k, v in taken:
        c.gather(0, rows, starts, k, v)
        assert torch.equal(k.cpu().view(torch.int16), want[0].view(torch.int16))
        assert torch.equal(v.cpu().view(torch.int16), want[1].view(torch.int16))
    crossing = wide.as_strided((n, heads, dim), (2 * dim, dim, 1), dim + 32)  # from one row to the next
    refused = [(other, other), (one[:n], one[n - 1:2 * n - 1]), (one[:n], one[0::2]), (one[1::2], one[n:]),
               (wide[:n, :, :dim], wide[:n, :, 8:dim + 8]), (wide[:n, :, dim:], crossing)]
    for t in _planes(c) + [c.slots, c.workspace]:
        m = of(t)
        if m.shape[0]:
            few = min(len(m), n)
            refused += [(m[:few], other[:few]), (other[:few], m[-few:])]
    both = torch.zeros(4096, dtype=torch.int32, device=gpu_device)  # outputs around rows and starts
    at = of(both)
    both[100:101], both[104:106] = rows, starts
    for k, v in refused:
        kept = k.clone(), v.clone()
        with pytest.raises(ValueError, match="share no memory"):
            c.gather(0, rows, starts if len(k) == n else _i32([0, len(k)], gpu_device), k, v)
        assert torch.equal(k.view(torch.int16), kept[0].view(torch.int16)) and torch.equal(v.view(torch.int16), kept[1].view(torch.int16))
    for a, b in ((both[100:101], starts), (rows, both[104:106])):
        for k, v in ((at[:n], other), (other, at[:n])):
            with pytest.raises(ValueError, match="share no memory"):
                c.gather(0, a, b, k, v)
    c.gather(0, both[100:101], both[104:106], at[n:2 * n], other)
    after = [_bytes(t) for t in _planes(c)] + [t.cpu() for t in (c.tables, c.lengths, c.refs, c.slots, c.starts)]
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    for stride in (1 << 31, (1 << 30) + 8):
        assert N.lib().kv_cache_gather(c._cache, 0, rows.data_ptr(), starts.data_ptr(), 1, one.data_ptr(), other.data_ptr(), stride,
                                       64, n, None) == N.MOE_EINVAL
    c.check_inputs()
