"""The paged key-value cache against its oracle: integers and bytes exactly
(MI355X only)."""
import random

import pytest
import torch

from llm_gpu_kernels_amd import PagedKVCache, _native as N
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


class Pair:
    """A cache and its oracle, every call made on both and compared."""

    def __init__(self, device, pages, page, sequences, max_pages, max_tokens, heads=2, dim=64, layers=2,
                 dtype=torch.bfloat16):
        self.device = device
        self.gpu = PagedKVCache(pages, page, heads, dim, sequences=sequences, max_pages=max_pages,
                                max_tokens=max_tokens, layers=layers, dtype=dtype, device=device)
        self.ref = S.Cache(pages, page, sequences, max_pages, max_tokens)
        g = torch.Generator().manual_seed(pages)
        self.k = torch.randn(self.gpu.k.shape, generator=g).to(dtype)
        self.v = torch.randn(self.gpu.k.shape, generator=g).to(dtype)
        self.gpu.k.copy_(self.k)
        self.gpu.v.copy_(self.v)

    def call(self, name, *lists, **kw):
        getattr(self.gpu, name)(*(_i32(x, self.device) for x in lists), **kw)
        getattr(self.ref, name)(*lists, **kw)
        for a, b in self.ref.moves:
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]

    def compare(self):
        c, r = self.gpu, self.ref
        assert c.lengths.tolist() == r.lengths
        assert c.refs.tolist() == r.refs
        assert c.tables.tolist() == [t + [-1] * (r.max_pages - len(t)) for t in r.tables]
        assert c.slots.tolist() == r.slots
        assert c.starts.tolist() == r.starts
        assert torch.equal(c.k.cpu().view(torch.int16), self.k.view(torch.int16))
        assert torch.equal(c.v.cpu().view(torch.int16), self.v.view(torch.int16))
        assert c.read_status() == r.status
        r.status = 0
        r.check()


@pytest.mark.parametrize("pages,page,sequences,max_pages,max_tokens,steps", [
    (40, 16, 6, 12, 200, 120),
    (1, 16, 1, 1, 16, 20),
    (300, 48, 70, 9, 1000, 60),       # more rows than a wave holds
    (9000, 16, 200, 60, 4000, 25),    # more pages than one scanned chunk
    (2100, 16, 1024, 8, 2048, 12),    # a row per thread of the planning workgroup
])
def test_random_calls(pages, page, sequences, max_pages, max_tokens, steps, gpu_device):
    rng = random.Random(pages)
    p = Pair(gpu_device, pages, page, sequences, max_pages, max_tokens, heads=1, layers=1 if pages > 1000 else 3)

    def rows(n):
        return [rng.randrange(-1, sequences + (rng.random() < 0.05)) for _ in range(min(n, sequences))]

    refused = 0
    for _ in range(steps):
        what = rng.choice(["reserve", "reserve", "step", "fork", "fork", "free", "compact"])
        if what == "reserve":
            few = max(1, max_tokens // sequences)
            p.call("reserve", [rng.choice([0, 0, 1, few, 2 * few]) for _ in range(sequences)])
        elif what == "step":
            counts = [int(n > 0 and rng.random() < 0.9) for n in p.ref.lengths]
            p.call("reserve", counts, stride=1)
        elif what == "fork":
            n = rng.randint(1, sequences)
            empty = [i for i, x in enumerate(p.ref.lengths) if x == 0]
            p.call("fork", rows(n), [rng.choice(empty) if empty and rng.random() < 0.9 else r for r in rows(n)])
        elif what == "free":
            p.call("free", rows(rng.randint(1, max(1, sequences // 2))))
        else:
            p.call("compact")
            assert p.gpu.used_pages.item() == sum(r > 0 for r in p.ref.refs)
        refused += bool(p.ref.status & (N.KV_STATUS_OUT_OF_PAGES | N.KV_STATUS_TOO_LONG))
        p.compare()


def test_copy_on_write(gpu_device):
    """Rows that share a partly filled page: each that grows gets a copy, the last
    of them keeps the page when all do; a full page is shared on."""
    p = Pair(gpu_device, 30, 16, 8, 4, 64, layers=3)
    p.call("reserve", [5, 0, 0, 0, 16, 0, 0, 0])
    p.call("fork", [0, 0, 4, 0], [1, 2, 5, 3])
    p.compare()
    p.call("reserve", [1, 0, 1, 0, 1, 1, 0, 0], stride=1)   # rows 1 and 3 keep the page
    assert len(p.ref.moves) == 2
    p.compare()
    p.call("reserve", [0, 3, 0, 20, 0, 0, 0, 0])            # both holders grow: one copy
    assert len(p.ref.moves) == 1
    p.compare()


def test_same_row_twice_and_bad_rows(gpu_device):
    p = Pair(gpu_device, 30, 16, 8, 4, 64)
    p.call("reserve", [20, 7, 0, 0, 0, 0, 0, 0])
    p.call("fork", [0, 1, 0, 8, 1, -1, 2], [2, 2, 3, 4, 1, 5, 6])  # 2 twice, 8 no row, 1 holds tokens, 2 is empty
    assert p.ref.status == N.KV_STATUS_BAD_ROW | N.KV_STATUS_NOT_EMPTY
    p.compare()
    p.call("free", [2, 2, 0, -1, 2, 8])
    assert p.ref.status == N.KV_STATUS_BAD_ROW
    p.compare()
    p.call("fork", [3, 7], [0, 2])   # a chain: row 2 is empty before and after
    p.call("fork", [3, 2], [2, 4])   # 2 is filled by this call, 4 reads it as it was: empty
    assert p.ref.lengths[4] == 0
    p.compare()


def test_refused_reserves_change_nothing(gpu_device):
    p = Pair(gpu_device, 6, 16, 3, 4, 80)
    p.call("reserve", [30, 17, 0])
    for counts, stride, status in [([0, 0, 64], 0, N.KV_STATUS_OUT_OF_PAGES), ([35, 0, 0], 0, N.KV_STATUS_TOO_LONG),
                                   ([0, -1, 0], 0, N.KV_STATUS_BAD_COUNT), ([3, 0, 0], 2, N.KV_STATUS_BAD_COUNT),
                                   ([1 << 30, 0, 0], 0, N.KV_STATUS_BAD_COUNT),
                                   ([30, 40, 30], 0, N.KV_STATUS_BAD_COUNT)]:
        p.call("reserve", counts, stride=stride)
        assert p.ref.status == status
        p.compare()
    with pytest.raises(ValueError):
        p.gpu.reserve(_i32([0, 0], gpu_device))
    with pytest.raises(ValueError):
        p.gpu.reserve(_i32([0, 0, 0], gpu_device), stride=27)
    with pytest.raises(ValueError):
        p.gpu.free(_i32([0, 0, 0, 0], gpu_device))
    with pytest.raises(ValueError):
        p.gpu.append(2, *(torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=gpu_device) for _ in range(2)))
    p.call("reserve", [0, 0, 32])
    p.compare()
    p.call("reserve", [0, 0, 1])
    with pytest.raises(RuntimeError, match="no room"):
        p.gpu.check_inputs()
    p.gpu.check_inputs()  # reported once


def test_bad_state_is_reported(gpu_device):
    """Lengths and page numbers that a program wrote wrongly: found, not followed."""
    for what in ("length", "long", "page"):
        p = Pair(gpu_device, 10, 16, 3, 4, 64)
        p.call("reserve", [20, 3, 0])
        if what == "page":
            p.gpu.tables[0, 1] = 1 << 20
        else:
            p.gpu.lengths[0] = -5 if what == "length" else 1000
        p.gpu.reserve(_i32([1, 1, 1], gpu_device))
        assert p.gpu.read_status() & N.KV_STATUS_BAD_STATE
        assert set(p.gpu.slots.tolist()) == {-1} and p.gpu.lengths[1:].tolist() == [3, 0]
        p.gpu.compact()
        assert p.gpu.read_status() & N.KV_STATUS_BAD_STATE
        p.gpu.fork(_i32([0], gpu_device), _i32([2], gpu_device))
        assert p.gpu.read_status() & N.KV_STATUS_BAD_STATE
        p.gpu.free(_i32([0, 2], gpu_device))
        assert p.gpu.read_status() & N.KV_STATUS_BAD_STATE
        assert p.gpu.lengths.tolist() == [0, 3, 0]


@pytest.mark.parametrize("dtype,heads,dim,page,fused", [
    (torch.bfloat16, 8, 128, 16, True), (torch.float16, 2, 64, 48, False), (torch.bfloat16, 1, 64, 16, False),
    (torch.float16, 3, 128, 32, True)])
def test_append(dtype, heads, dim, page, fused, gpu_device):
    """Rows of tokens land in their slots of their layer; everything else stays."""
    p = Pair(gpu_device, 40, page, 5, 8, 300, heads, dim, 3, dtype)
    p.call("reserve", [page * 2 + 3, 0, 1, 17, page])
    n = sum([page * 2 + 3, 0, 1, 17, page])
    for layer, tokens in ((1, n), (2, n - 5), (0, 300), (0, 0)):
        rows = torch.randn(tokens, 2 * heads + 1, dim).to(dtype).to(gpu_device)
        k, v = (rows[:, 1:1 + heads], rows[:, 1 + heads:]) if fused else (rows[:, :heads].contiguous(),
                                                                          rows[:, heads:2 * heads].contiguous())
        p.gpu.append(layer, k, v)
        for i, slot in enumerate(p.ref.slots[:tokens]):
            if slot >= 0:
                p.k[layer, slot // page, :, slot % page] = k[i].cpu()
                p.v[layer, slot // page, :, slot % page] = v[i].cpu()
        p.compare()


def test_append_one_token_of_odd_strides(gpu_device):
    """A single token whose strides torch leaves arbitrary, and slots that a
    program set outside the cache."""
    p = Pair(gpu_device, 4, 16, 1, 4, 8, heads=1)
    k = torch.randn(1, 1, 64, device=gpu_device).to(torch.bfloat16).as_strided((1, 1, 64), (3, 5, 1))
    p.gpu.slots.copy_(torch.tensor([40, 64, -7, 1 << 40, 63, -1, -1, -1], device=gpu_device))
    p.gpu.append(1, k, k)
    many = torch.randn(5, 1, 64, device=gpu_device).to(torch.bfloat16)
    p.gpu.append(0, many, many)
    for kv, ours in ((p.gpu.k, p.k), (p.gpu.v, p.v)):
        ours[1, 2, 0, 8] = k[0, 0].cpu()
        ours[0, 2, 0, 8], ours[0, 3, 0, 15] = many[0, 0].cpu(), many[4, 0].cpu()
        assert torch.equal(kv.cpu().view(torch.int16), ours.view(torch.int16))


def test_call_refusals(gpu_device):
    """Arguments that the host can check are refused before anything is enqueued."""
    p = Pair(gpu_device, 4, 16, 2, 2, 8, heads=2)
    ok = torch.zeros(8, 2, 64, dtype=torch.bfloat16, device=gpu_device)
    rows = torch.zeros(2, dtype=torch.int32, device=gpu_device)
    for layer in (-1, 2, 2 ** 32, 1.0, None):
        with pytest.raises(ValueError, match="layer"):
            p.gpu.append(layer, ok, ok)
    for k in (ok[:7], ok[:, :1], ok.half(), ok.cpu(), ok[:, :, ::2], torch.cat([ok, ok]), ok[0]):
        with pytest.raises(ValueError):
            p.gpu.append(0, k, ok)
    with pytest.raises(ValueError, match="max_tokens"):
        p.gpu.append(0, torch.cat([ok, ok]), torch.cat([ok, ok]))
    with pytest.raises(ValueError):
        p.gpu.append(0, ok.transpose(0, 1).contiguous().transpose(0, 1), ok)
    for counts, stride in ((rows[:1], 0), (rows.cpu(), 0), (rows, -1), (rows, 5), (rows, 1.0)):
        with pytest.raises(ValueError):
            p.gpu.reserve(counts, stride)
    with pytest.raises(TypeError):
        p.gpu.reserve(rows.long())
    for src, dst in ((rows, rows[:1]), (torch.cat([rows, rows]), torch.cat([rows, rows])), (rows[None], rows[None])):
        with pytest.raises(ValueError):
            p.gpu.fork(src, dst)
    assert p.gpu.read_status() == 0 and torch.equal(p.gpu.k.cpu(), p.k) and not p.gpu.refs.any()


def test_captured_steps(gpu_device):
    """A captured decode step (reserve and append) replayed on another stream,
    with eager forks and frees between, matches the oracle; so do captured
    frees, forks and compactions."""
    p = Pair(gpu_device, 60, 16, 6, 6, 96, heads=2, layers=2)
    p.call("reserve", [10, 16, 0, 33, 0, 0])
    counts, src, dst, rows = (_i32(x, gpu_device) for x in ([1, 1, 0, 1, 0, 0], [0, 3], [2, 4], [2, 4]))
    kv = torch.zeros(6, 4, 64, dtype=torch.bfloat16, device=gpu_device)
    side = torch.cuda.Stream(device=gpu_device)
    torch.cuda.synchronize()
    step, branch = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(step, stream=side):
        p.gpu.reserve(counts, stride=1)
        p.gpu.append(0, kv[:, :2], kv[:, 2:])
    with torch.cuda.graph(branch, stream=side):
        p.gpu.free(rows)
        p.gpu.compact()
        p.gpu.fork(src, dst)
    for i in range(6):
        kv.copy_(torch.randn(6, 4, 64))
        active = [1, 1, 0, 1, 0, 0] if i % 2 else [1, 0, 1, 1, 1, 0]
        counts.copy_(_i32(active, gpu_device))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            branch.replay()
            step.replay()
        torch.cuda.current_stream().wait_stream(side)
        for name, lists in (("free", [[2, 4]]), ("compact", []), ("fork", [[0, 3], [2, 4]])):
            getattr(p.ref, name)(*lists)
            for a, b in p.ref.moves:
                p.k[:, b], p.v[:, b] = p.k[:, a].clone(), p.v[:, a].clone()
        p.ref.reserve(active, stride=1)
        for a, b in p.ref.moves:
            p.k[:, b], p.v[:, b] = p.k[:, a].clone(), p.v[:, a].clone()
        for row, slot in enumerate(p.ref.slots[:6]):
            if slot >= 0:
                p.k[0, slot // 16, :, slot % 16] = kv[row, :2].cpu()
                p.v[0, slot // 16, :, slot % 16] = kv[row, 2:].cpu()
        p.compare()
        if i == 3:
            p.call("free", [1])
            p.call("reserve", [0, 9, 0, 0, 0, 0])
            p.compare()


def test_large_pages_and_offsets(gpu_device):
    """Page offsets past 2^32 bytes: pages copied, moved and written at the far end
    of a cache of 9 GiB."""
    pages, page, heads, dim = 18000, 64, 32, 128
    c = PagedKVCache(pages, page, heads, dim, sequences=4, max_pages=pages, max_tokens=256, device=gpu_device)
    assert c.k.numel() * 2 > 1 << 33
    last = pages - 2
    c.refs[:last] = 1                       # someone else's: only the two last pages are free
    c.reserve(_i32([5, 0, 0, 0], gpu_device))
    row = torch.randn(5, heads, dim, device=gpu_device).to(torch.bfloat16)
    c.append(0, row, -row)
    c.fork(_i32([0], gpu_device), _i32([1], gpu_device))
    c.reserve(_i32([0, 1, 0, 0], gpu_device))
    assert c.tables[:2, 0].tolist() == [last, last + 1] and c.read_status() == 0
    for p in (last, last + 1):
        assert torch.equal(c.k[0, p, :, :5], row.transpose(0, 1)) and torch.equal(c.v[0, p, :, :5], -row.transpose(0, 1))
    c.refs[:last] = 0
    c.compact()
    assert c.tables[:2, 0].tolist() == [0, 1] and c.read_status() == 0 and c.used_pages.item() == 2
    for p in (0, 1):
        assert torch.equal(c.k[0, p, :, :5], row.transpose(0, 1)) and torch.equal(c.v[0, p, :, :5], -row.transpose(0, 1))


def test_as_many_pages_and_tokens_as_allowed(gpu_device):
    """2^20 pages, all but some at the end in use, and a reserve of 2^20 tokens."""
    pages, tokens = N.KV_MAX_PAGES, N.KV_MAX_TOKENS
    c = PagedKVCache(pages, 16, 1, 64, sequences=3, max_pages=pages, max_tokens=tokens, device=gpu_device)
    c.refs[:pages - 70000] = 1
    c.reserve(_i32([tokens - 1000, 0, 1000], gpu_device))
    need = [-(-(tokens - 1000) // 16), 0, 63]
    first = pages - 70000
    assert c.read_status() == 0 and c.lengths.tolist() == [tokens - 1000, 0, 1000]
    ids = torch.arange(first, first + sum(need), dtype=torch.int32, device=gpu_device)
    assert torch.equal(c.tables[0, :need[0]], ids[:need[0]]) and torch.equal(c.tables[2, :63], ids[need[0]:])
    at = torch.arange(tokens, device=gpu_device)
    row_start = torch.where(at < tokens - 1000, 0, tokens - 1000)
    page = torch.where(at < tokens - 1000, first, first + need[0]) + (at - row_start) // 16
    assert torch.equal(c.slots, page * 16 + (at - row_start) % 16)
    c.refs[:first] = 0
    c.refs[5] = 1
    c.k[0, first + 3].fill_(3.0)
    c.compact()
    assert c.read_status() == 0 and c.used_pages.item() == sum(need) + 1
    # Pages below the count that are free, in order, took the used ones from it on.
    free = torch.tensor([p for p in range(sum(need) + 1) if p != 5], device=gpu_device)
    assert torch.equal(c.tables[0, :need[0]].long(), free[:need[0]]) and (c.k[0, free[3]] == 3).all()
    assert c.refs[:sum(need) + 1].min() == 1 and c.refs[sum(need) + 1:].max() == 0
