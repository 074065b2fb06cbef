"""Decode attention where groups of sequences start with the same keys, against attention
in 64 bits of every sequence by its own table (MI355X only).  Tolerances: oracle/
serving_oracle.py, tolerance(); the two parts of a row are joined in fp32."""
import ctypes

import pytest
import torch

from llm_gpu_kernels_amd import PagedKVCache, _native as N, prepare_paged_gqa, prepare_shared_gqa
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu

HEADS = [(32, 8, 128), (8, 8, 128), (12, 4, 64), (14, 2, 64), (6, 6, 64), (16, 1, 128), (40, 2, 128), (64, 1, 64)]
TYPES = [torch.bfloat16, torch.float16]


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _assert_close(out, ref, bound, keys, vmax):
    off = (out.double().cpu() - ref).abs()
    tol = S.tolerance(ref, bound, out.dtype, keys, vmax)
    assert torch.isfinite(out).all()
    worst = (off / tol.clamp(min=1e-30)).max().item()
    assert worst <= 1.0, worst


@pytest.fixture(autouse=True, params=["narrow", "wide"])
def tables(request, monkeypatch):
    """Tables just wide enough, of which small ones are worked on row by row, and wide
    ones, whose groups are worked on together."""
    monkeypatch.setattr(Groups, "least_width", 1 if request.param == "narrow" else 1000)


class Groups:
    """Groups as (prefix, lengths of the members), sequences of no group before and behind
    them.  Whole pages of a prefix are held once, the rest of it by every member; places
    behind each sequence's end hold NaN, table entries behind the last page an impossible
    number."""

    least_width = 1

    def __init__(self, groups, hq, hkv, d, page, dtype, device, before=(), behind=(), order="heads"):
        self.device = device
        self.lengths = list(before) + [n for _, members in groups for n in members] + list(behind)
        g = torch.Generator().manual_seed(sum(self.lengths) + page + hq)
        owner = [None] * len(before) + [i for i, (_, m) in enumerate(groups) for _ in m] + [None] * len(behind)
        plans, count = [], 0  # pages by number in order of use
        shared = []
        for prefix, members in groups:
            whole = min([prefix] + [n for n in members if n > 0]) // page
            shared.append(list(range(count, count + whole)))
            count += whole
        for n, o in zip(self.lengths, owner):
            start = shared[o] if o is not None and n > 0 else []
            own = max(0, -(-n // page) - len(start))
            plans.append(start + list(range(count, count + own)))
            count += own
        count += 3
        perm = torch.randperm(count, generator=g).tolist()
        shape = (count, hkv, page, d)
        kv = [torch.randn(shape, generator=g) for _ in range(2)]
        kv = [t.to(dtype) for t in kv]
        width = max([len(x) for x in plans] + [self.least_width]) + 2
        self.tables = [[perm[i] for i in x] + [1 << 29] * (width - len(x)) for x in plans]
        heads_of = {}
        for b, (n, o) in enumerate(zip(self.lengths, owner)):
            if o is None or n == 0:
                continue
            at = len(shared[o])
            rest = min([groups[o][0]] + [m for m in groups[o][1] if m > 0]) - at * page
            if rest > 0:  # the page that a member has of its own, from the others' first
                if o in heads_of:
                    for t in kv:
                        t[self.tables[b][at], :, :rest] = t[self.tables[heads_of[o]][at], :, :rest]
                heads_of.setdefault(o, b)
        for n, row in zip(self.lengths, self.tables):
            if n % page:
                for t in kv:
                    t[row[n // page], :, n % page:] = float("nan")
        for t in kv:
            t[perm[count - 3:]] = float("nan")
        self.starts = [len(before)]
        for _, members in groups:
            self.starts.append(self.starts[-1] + len(members))
        self.prefixes = [p for p, _ in groups]
        self.q = torch.randn(len(self.lengths), hq, d, generator=g).to(dtype).to(device)
        if order == "tokens":
            kv = [t.transpose(1, 2).contiguous().to(device).transpose(1, 2) for t in kv]
        self.k, self.v = (t.to(device) for t in kv)
        self.gt, self.gl = _i32(self.tables, device), _i32(self.lengths, device)
        self.gs, self.gp = _i32(self.starts, device), _i32(self.prefixes, device)

    def plan(self, **kw):
        return prepare_shared_gqa(self.q, self.k, self.v, self.gt, self.gl, self.gs, self.gp, **kw)

    def check(self, plan, scale=None, status=0):
        ref, bound = S.paged_attention(self.q.cpu(), self.k.cpu(), self.v.cpu(), self.tables, self.lengths, scale)
        _assert_close(plan.output, ref, bound, max(self.lengths), self.v.float().nan_to_num(0).abs().max().item())
        for b, n in enumerate(self.lengths):
            if n == 0:
                assert (plan.output[b] == 0).all()
        assert plan.read_status() == status


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_heads(hq, hkv, d, dtype, gpu_device):
    x = Groups([(100, [120, 100, 133]), (37, [60, 0, 41, 37, 300])], hq, hkv, d, 16, dtype, gpu_device, before=[50],
               behind=[0, 77])
    x.check(x.plan())


@pytest.mark.parametrize("groups,before,behind,page", [
    ([(16, [17, 17])], [], [], 16),
    ([(15, [17, 17])], [], [], 16),                    # no whole block: nothing is shared
    ([(1, [1, 1, 1])], [], [], 16),
    ([(48, [48, 48])], [], [], 48),                    # no keys behind the prefix
    ([(64, [64, 64, 65])], [], [], 16),
    ([(500, [40, 700])], [], [], 16),                  # the shortest member bounds it
    ([(300, [400])], [5], [], 16),                     # one member
    ([(300, [400, 0, 0])], [5], [], 16),               # one member that has keys
    ([(300, [0, 0]), (0, [30, 40]), (200, [220, 230])], [], [9], 32),
    ([(1000, [1003, 1100]), (1024, [1030, 1024, 2100])], [], [], 1024),
    ([(170, [171 + i % 5 for i in range(90)])], [3], [], 80),   # more rows than a workgroup's
    ([(33 + i, [60 + i, 70 + i]) for i in range(150)], [], [], 16),
    ([(5000, [5100, 5020, 5333])], [], [4000], 32),
    ([(40, [50 + i % 9 for i in range(700)])], [], [], 16),
    ([], [10, 20], [], 16),
], ids=lambda x: str(x)[:28])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_groups(groups, before, behind, page, order, gpu_device):
    x = Groups(groups, 8, 2, 128, page, torch.bfloat16, gpu_device, before, behind, order)
    x.check(x.plan())


def test_one_kv_head_of_many_rows(gpu_device):
    """64 query heads of one KV head: 30 members are 1920 rows, eight tiles."""
    x = Groups([(200, [210 + i for i in range(30)]), (64, [90, 100])], 64, 1, 64, 16, torch.float16, gpu_device)
    x.check(x.plan(scale=0.2), 0.2)


def test_long_prefix(gpu_device):
    x = Groups([(20011, [20040, 20500, 20012, 21000])], 8, 2, 128, 16, torch.bfloat16, gpu_device)
    x.check(x.plan())


def test_many_sequences(gpu_device):
    """More sequences than the planning workgroup holds, most of them in no group."""
    x = Groups([(30, [40, 33])] * 40, 2, 1, 64, 16, torch.bfloat16, gpu_device, before=[i % 7 for i in range(5000)],
               behind=[i % 5 for i in range(4000)])
    x.check(x.plan())


@pytest.mark.parametrize("groups,members,behind", [(64, 4, 0), (64, 4, 1), (65, 3, 0), (1024, 2, 3)])
def test_many_groups(groups, members, behind, gpu_device):
    """About and past what every workgroup plans by itself, and as many as a call allows."""
    x = Groups([(33 + i % 20, [40 + (i + 7 * j) % 30 for j in range(members)]) for i in range(groups)], 2, 1, 64, 16,
               torch.bfloat16, gpu_device, behind=[50] * behind)
    x.check(x.plan())


def test_every_prefix_length(gpu_device):
    """One set of tensors, starts and prefixes changed between runs."""
    x = Groups([(160, [161 + 3 * i for i in range(12)])], 8, 2, 128, 16, torch.bfloat16, gpu_device, before=[40], behind=[50])
    plan = x.plan()
    for prefix in (0, 1, 15, 16, 17, 31, 32, 47, 160, 161, 10 ** 6, 2 ** 31 - 1):
        x.gp[0] = prefix
        if prefix <= 161:
            plan.run()
            x.check(plan)
    x.gp[0] = 2 ** 31 - 1   # 161 keys: the shortest member's 161st is its own, and outside the whole blocks
    plan.run()
    x.check(plan)
    x.gp[0] = 160
    for starts in ([1, 13], [3, 9], [5, 5], [12, 13], [1, 1]):
        x.gs.copy_(_i32(starts, gpu_device))
        plan.run()
        x.check(plan)


@pytest.mark.parametrize("starts", [[5, 3, 9], [-1, 4, 9], [0, 4, 10], [0, 2 ** 31 - 1, 9], [-2 ** 31, 0, 2 ** 31 - 1]])
def test_bad_starts(starts, gpu_device):
    """Reported; every sequence is attended by itself."""
    x = Groups([(64, [70, 80, 90]), (96, [99, 100, 130, 140, 150, 160])], 8, 2, 128, 16, torch.bfloat16, gpu_device)
    plan = x.plan()
    x.check(plan)
    x.gs.copy_(_i32(starts, gpu_device))
    plan.run()
    x.check(plan, status=N.GQA_STATUS_BAD_BOUNDS)
    x.gs.copy_(_i32(x.starts, gpu_device))
    x.gp[1] = -5
    plan.run()
    x.check(plan, status=N.GQA_STATUS_BAD_BOUNDS)


def test_bad_pages_and_lengths(gpu_device):
    x = Groups([(64, [70, 80, 90]), (48, [60, 61])], 8, 2, 128, 16, torch.bfloat16, gpu_device)
    plan = x.plan()
    clean = plan.output.clone()
    for bad in (-1, x.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        x.gt[:3, 1] = bad     # keys 16 to 31 of the first group
        out = plan.run()
        assert plan.read_status() == N.GQA_STATUS_BAD_PAGE and plan.read_status() == 0
        assert torch.equal(out[3:], clean[3:])
        for b in range(3):
            keys = [(x.tables[b][j // 16], j % 16) for j in range(x.lengths[b]) if j // 16 != 1]
            rows = torch.tensor([p for p, _ in keys]), torch.tensor([r for _, r in keys])
            ref, bound = S.attention_rows(x.q[b].cpu(), x.k.cpu()[rows[0], :, rows[1]], x.v.cpu()[rows[0], :, rows[1]])
            _assert_close(out[b], ref, bound, 90, 6.0)
    x.gt[:3] = -1
    assert (plan.run()[:3] == 0).all() and plan.read_status() == N.GQA_STATUS_BAD_PAGE
    x.gt.copy_(_i32(x.tables, gpu_device))
    x.gl[1] = -3              # out of the group, like an empty one
    out = plan.run()
    assert (out[1] == 0).all() and plan.read_status() == N.GQA_STATUS_BAD_BOUNDS
    lengths, x.lengths = x.lengths, [70, 0, 90, 60, 61]
    ref, bound = S.paged_attention(x.q.cpu(), x.k.cpu(), x.v.cpu(), x.tables, x.lengths)
    _assert_close(out, ref, bound, 90, 6.0)


def test_not_finite(gpu_device):
    """A NaN key of a prefix reaches its head of all members; an infinite value its dim."""
    x = Groups([(64, [70, 80, 90]), (64, [70, 100])], 8, 2, 128, 16, torch.bfloat16, gpu_device, behind=[33])
    plan = x.plan()
    clean = plan.output.clone()
    x.k[x.tables[0][2], 1, 5, 9] = float("nan")
    x.v[x.tables[3][0], 0, 3, 100] = float("inf")
    out = plan.run()
    assert out[:3, 4:].isnan().all() and torch.equal(out[:3, :4], clean[:3, :4])
    assert (out[3:5, :4, 100] == float("inf")).all() and torch.isfinite(out[3:5, :4, :100]).all()
    assert torch.equal(out[3:5, 4:], clean[3:5, 4:]) and torch.equal(out[5], clean[5])


def test_large_scores(gpu_device):
    """Maxima that differ by far between the prefix and the rest."""
    x = Groups([(96, [120, 130])], 8, 2, 128, 16, torch.float16, gpu_device)
    x.k[x.tables[0][1]] *= 8
    x.k[x.tables[1][7]] *= 16
    plan = x.plan()
    ref, bound = S.paged_attention(x.q.cpu(), x.k.cpu(), x.v.cpu(), x.tables, x.lengths)
    # Scores of up to 16 times as much are off by 16 times as much: 2^-9 + 2^-12 of the bound.
    off = (plan.output.double().cpu() - ref).abs()
    tol = S.tolerance(ref, bound, torch.float16, 130, 5.0) + bound * 2.0 ** -8
    assert (off <= tol).all()


def test_offsets_past_32_bits(gpu_device):
    x = Groups([(1000, [1040, 1025, 1500])], 16, 8, 128, 128, torch.bfloat16, gpu_device)
    used, count = x.k.shape[0], 20000
    big = []
    where = [count - 1 - 2 * i if i % 2 else 3 * i for i in range(used)]
    for t in (x.k, x.v):
        y = torch.empty((count,) + t.shape[1:], dtype=t.dtype, device=gpu_device)
        assert y.numel() * 2 > 1 << 32
        y[torch.tensor(where, device=gpu_device)] = t
        big.append(y)
    tables = [[where[p] if p < used else p for p in row] for row in x.tables]
    plan = prepare_shared_gqa(x.q, *big, _i32(tables, gpu_device), x.gl, x.gs, x.gp)
    x.check(plan)


def test_keys_up_to_2_31(gpu_device):
    """The longest sequences that a call allows, of one page over and over: attention over its
    16 keys, but that the second sequence lacks the last page's last 5.  A workgroup has some 2^17
    stages of the prefix, so its denominators are off by 2^17 * 2^-24 of themselves, and O, of two
    products a stage, by 2^-6 of the bound; the 5 keys are 2^-28 of all."""
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(1, 1, 16, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(2, 4, 64, generator=g).to(torch.bfloat16)
    pages = 2 ** 27 - 1
    tables = torch.zeros(2, pages, dtype=torch.int32, device=gpu_device)
    lengths = _i32([16 * pages, 16 * pages - 5], gpu_device)
    plan = prepare_shared_gqa(q.to(gpu_device), k.to(gpu_device), v.to(gpu_device), tables, lengths, _i32([0, 2], gpu_device),
                              _i32([2 ** 31 - 1], gpu_device))
    plan.check_inputs()
    ref, bound = S.paged_attention(q, k, v, [[0], [0]], [16, 16])
    off, tol = (plan.output.double().cpu() - ref).abs(), S.tolerance(ref, bound, torch.bfloat16, 16, 6.0)
    assert (off <= tol + bound * (2.0 ** -6 + 2.0 ** -7 + 2.0 ** -12)).all()


def test_two_streams_and_a_graph(gpu_device):
    a = Groups([(640, [700, 650, 2000])], 8, 2, 128, 16, torch.bfloat16, gpu_device, behind=[50])
    b = Groups([(64, [70, 80, 90]), (96, [99, 100])], 8, 2, 128, 16, torch.bfloat16, gpu_device)
    pa, pb = a.plan(), b.plan()
    want_a, want_b = pa.output.clone(), pb.output.clone()
    sa, sb, graph = torch.cuda.Stream(gpu_device), torch.cuda.Stream(gpu_device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=sa):
        pa.run()
    for i in range(5):
        pa.output.zero_()
        pb.output.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(sa):
            graph.replay()
        with torch.cuda.stream(sb):
            pb.run()
        torch.cuda.synchronize()
        assert torch.equal(pa.output, want_a) and torch.equal(pb.output, want_b)
    a.lengths[1] = 645  # the graph reads lengths, starts and prefixes when it is replayed
    a.gl[1] = 645
    a.gp[0] = 100
    graph.replay()
    torch.cuda.synchronize()
    a.check(pa)


def test_forked_samples(gpu_device):
    """Prompts forked into samples that grow by tokens of their own."""
    g = torch.Generator().manual_seed(4)
    hq, hkv, d, page = 8, 2, 128, 16
    c = PagedKVCache(200, page, hkv, d, sequences=9, max_pages=30 * Groups.least_width, max_tokens=400, device=gpu_device)
    counts = [150, 0, 0, 0, 77, 0, 0, 20, 0]
    c.reserve(_i32(counts, gpu_device))
    rows = torch.randn(400, 2 * hkv, d, generator=g).to(torch.bfloat16).to(gpu_device)
    c.append(0, rows[:247, :hkv], rows[:247, hkv:])
    c.fork(_i32([0, 0, 0, 4, 4], gpu_device), _i32([1, 2, 3, 5, 6], gpu_device))
    lengths = [150, 150, 150, 150, 77, 77, 77, 20, 0]
    starts, prefixes = _i32([0, 4, 7], gpu_device), _i32([150, 77], gpu_device)
    q = torch.randn(9, hq, d, generator=g).to(torch.bfloat16).to(gpu_device)
    plan = prepare_shared_gqa(q, c.k[0], c.v[0], c.tables, c.lengths, starts, prefixes)
    alone = prepare_paged_gqa(q, c.k[0], c.v[0], c.tables, c.lengths)
    for step in range(40):
        grow = [int(n > 0 and (step + b) % 4 > 0) for b, n in enumerate(lengths)]
        c.reserve(_i32(grow, gpu_device), stride=1)
        lengths = [n + x for n, x in zip(lengths, grow)]
        new = torch.randn(9, 2 * hkv, d, generator=g).to(torch.bfloat16).to(gpu_device)
        c.append(0, new[:, :hkv], new[:, hkv:])
        plan.run()
        alone.run()
        if step % 8 == 7:
            ref, bound = S.paged_attention(q.cpu(), c.k[0].cpu(), c.v[0].cpu(), c.tables.tolist(), lengths)
            for out in (plan.output, alone.output):
                _assert_close(out, ref, bound, 200, 6.0)
        if step == 20:
            c.compact()
    plan.check_inputs()
    c.check_inputs()


def test_nothing_to_do(gpu_device):
    x = Groups([(64, [70, 80])], 8, 2, 128, 16, torch.bfloat16, gpu_device)
    empty = prepare_shared_gqa(x.q[:0], x.k, x.v, x.gt[:0], x.gl[:0], x.gs[:1], x.gp[:0])
    assert empty.run().shape == (0, 8, 128)
    x.gl.zero_()
    plan = x.plan()
    assert (plan.run() == 0).all() and plan.read_status() == 0


@pytest.mark.parametrize("lengths,kept", [([64, 64, -3], [64, 64, 0]), ([-2 ** 31, 64, 64], [0, 64, 64]),
                                          ([-1, -2, -3], [0, 0, 0]), (["past"] * 3, ["table"] * 3),
                                          ([2 ** 31 - 1, "table", "past"], ["table"] * 3)], ids=str)
@pytest.mark.parametrize("groups,members", [(1, 3), (65, 3), (1, 258)], ids=["here", "groups", "rows"])
def test_bad_lengths_without_keys_behind_a_prefix(groups, members, lengths, kept, gpu_device):
    """Lengths out of range are reported where every key is one of a prefix too, planned by each
    workgroup and (more than 64 groups or 256 sequences) by a launch before, and are worked on as
    if they were at the limit that they pass."""
    g = torch.Generator().manual_seed(groups + members)
    page, hq, hkv, d, width = 16, 2, 1, 64, 4 if Groups.least_width == 1 else 600
    table = page * width
    numbers = {"past": table + 1, "table": table}
    lengths, kept = ([numbers.get(n, n) for n in x] for x in (lengths, kept))
    # The bad group last, its third length that of all members behind; the others of 32 keys.
    before = (groups - 1) * members
    lengths = [32] * before + lengths + lengths[2:] * (members - 3)
    kept = [32] * before + kept + kept[2:] * (members - 3)
    rows = [[j % 40 for j in range(width)]] * len(lengths)  # 40 pages over and over
    k, v = (torch.randn(40, hkv, page, d, generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(len(lengths), hq, d, generator=g).to(torch.bfloat16)
    starts, prefixes = [i * members for i in range(groups + 1)], [32] * (groups - 1) + [table]
    args = [q.to(gpu_device), k.to(gpu_device), v.to(gpu_device), _i32(rows, gpu_device)]
    good = prepare_shared_gqa(*args, _i32(kept, gpu_device), _i32(starts, gpu_device), _i32(prefixes, gpu_device))
    assert good.read_status() == 0
    plan = prepare_shared_gqa(*args, _i32(lengths, gpu_device), _i32(starts, gpu_device), _i32(prefixes, gpu_device))
    for _ in range(2):
        assert plan.read_status() == N.GQA_STATUS_BAD_BOUNDS and plan.read_status() == 0
        assert torch.equal(plan.output, good.output)
        plan.run()
    ref, bound = S.paged_attention(q, k, v, rows, kept)
    _assert_close(good.output, ref, bound, table, 6.0)


def test_prefixes_longer_than_every_member(gpu_device):
    """Prefixes past the shortest member, up to the largest number: it bounds what is shared."""
    x = Groups([(160, [161 + 3 * i for i in range(12)])], 8, 2, 128, 16, torch.bfloat16, gpu_device, before=[40], behind=[50])
    plan = x.plan()
    for prefix in (161, 176, 10 ** 6, 2 ** 31 - 1):
        x.gp[0] = prefix
        plan.output.zero_()
        plan.run()
        x.check(plan)


def test_workspace(gpu_device):
    """Where every row goes by itself the status words are all that a plan needs, and less than
    what is asked for is refused."""
    x = Groups([(64, [70, 80, 90]), (48, [60, 61])], 8, 2, 128, 16, torch.bfloat16, gpu_device, behind=[33])
    plan = x.plan()
    assert (plan.workspace.numel() == 256) == (Groups.least_width == 1)
    x.check(plan)
    size, handle = ctypes.c_size_t(0), ctypes.c_void_p()
    d = plan._desc
    N.check(N.lib().gqa_shared_workspace_bytes(ctypes.byref(d), 2, ctypes.byref(size)), "size")
    assert size.value == plan.workspace.numel()
    d.workspace_bytes = size.value - 1
    assert N.lib().gqa_shared_plan_create(ctypes.byref(handle), ctypes.byref(d), 2, x.gs.data_ptr(), x.gp.data_ptr()) == N.MOE_ESPACE
    assert not handle.value
