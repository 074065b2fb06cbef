"""Device state of plans and caches that a program reads or wrote wrongly:
status words beside other streams, tables that name free pages, the largest
lengths (MI355X only)."""
import pytest
import torch

from llm_gpu_kernels_amd import PagedKVCache, _native as N, prepare_paged_gqa

pytestmark = pytest.mark.gpu


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def test_status_beside_another_stream(gpu_device):
    """A bit that a run on another stream latches while the word is read is in this
    reading or in the next."""
    q = torch.zeros(1, 1, 64, dtype=torch.float16, device=gpu_device)
    pages = torch.zeros(1, 1, 16, 64, dtype=torch.float16, device=gpu_device)
    tables, lengths = _i32([[0]], gpu_device), _i32([16], gpu_device)
    plan = prepare_paged_gqa(q, pages, pages, tables, lengths)
    side = torch.cuda.Stream(device=gpu_device)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda._sleep(1000)
    start.record()
    torch.cuda._sleep(1000000)
    end.record()
    torch.cuda.synchronize()
    per_us = 1000000 / (start.elapsed_time(end) * 1e3)
    lost = []
    for i in range(300):
        tables.fill_(7)
        plan.run()                                    # latches the page
        tables.fill_(0)
        lengths.fill_(17)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(max(1, int(i * 0.2 * per_us)))
            plan.run()                                # latches the length, 0 to 60 us later
        flags = plan.read_status()
        side.synchronize()
        flags |= plan.read_status()
        if flags != N.GQA_STATUS_BAD_PAGE | N.GQA_STATUS_BAD_BOUNDS:
            lost.append(i)
        lengths.fill_(16)
    assert not lost
    assert plan.read_status() == 0


@pytest.mark.parametrize("earlier", [False, True])
def test_compact_finds_free_pages_in_tables(earlier, gpu_device):
    """A table that names a free page behind those in use: reported, and left as it is
    instead of led to another row's page, whatever an earlier compaction moved."""
    c = PagedKVCache(20, 16, 1, 64, sequences=4, max_pages=4, max_tokens=256, device=gpu_device)
    c.reserve(_i32([64, 64, 64, 0], gpu_device))          # pages 0 to 11
    if earlier:
        c.free(_i32([0], gpu_device))
        c.compact()                                       # 8 to 11 go to 0 to 3
        assert c.tables[2].tolist() == [0, 1, 2, 3]
    for page in (9, 11, 12, 19):
        if not earlier and page < 12:
            continue
        before = c.tables.clone()
        c.tables[1, 2] = page
        c.compact()
        assert c.read_status() == N.KV_STATUS_BAD_STATE
        assert c.tables[1, 2].item() == page
        c.tables[1, 2] = before[1, 2]
        assert torch.equal(c.tables, before)
    c.compact()
    assert c.read_status() == 0


def test_largest_row_of_a_cache(gpu_device):
    """A row whose length in tokens, rounded up to pages, passes 2^31."""
    page, width = 1008, 2130440                           # page * width + page - 1 > 2^31
    c = PagedKVCache(4, page, 1, 64, sequences=2, max_pages=width, max_tokens=16, device=gpu_device)
    c.tables[0] = 1
    c.lengths[0] = page * width
    c.refs[1] = width
    c.fork(_i32([0], gpu_device), _i32([1], gpu_device))
    assert c.lengths.tolist() == [page * width] * 2 and c.refs.tolist() == [0, 2 * width, 0, 0]
    assert (c.tables == 1).all()
    c.reserve(_i32([1, 0], gpu_device))
    assert c.read_status() == N.KV_STATUS_TOO_LONG
    c.compact()
    assert (c.tables == 0).all() and c.refs.tolist() == [2 * width, 0, 0, 0]
    c.free(_i32([0, 1], gpu_device))
    assert c.read_status() == 0 and not c.refs.any() and not c.lengths.any() and (c.tables == -1).all()
