"""Packed prompt attention and paged decode attention against attention in 64
bits (MI355X only).  Tolerances: oracle/serving_oracle.py, tolerance()."""
import pytest
import torch

from llm_gpu_kernels_amd import PagedKVCache, _native as N, prepare_packed_gqa, prepare_paged_gqa
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu

HEADS = [(32, 8, 128), (8, 8, 128), (12, 4, 64), (14, 2, 64), (6, 6, 64), (16, 1, 128), (40, 2, 128), (64, 1, 64)]
TYPES = [torch.bfloat16, torch.float16]
# Tables of decode attention: just wide enough, wide, wide with a long last sequence.
# (Three ways in which the work is shared out.)
WIDE = ["narrow", "wide", "long"]


def _assert_close(out, ref, bound, keys, vmax):
    off = (out.double().cpu() - ref).abs()
    tol = S.tolerance(ref, bound, out.dtype, keys, vmax)
    assert torch.isfinite(out).all()
    worst = (off / tol.clamp(min=1e-30)).max().item()
    assert worst <= 1.0, worst


# ---- packed prompts ---------------------------------------------------------------


def _starts(lengths, first=0):
    out = [first]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _packed(lengths, hq, hkv, d, dtype, device, fused=False, first=0, behind=0, seed=0):
    g = torch.Generator().manual_seed(seed + sum(lengths))
    n = first + sum(lengths) + behind
    rows = torch.randn(n, hq + 2 * hkv, d, generator=g).to(dtype).to(device)
    q, k, v = rows.split([hq, hkv, hkv], dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    starts = _starts(lengths, first)
    return q, k, v, starts, torch.tensor(starts, dtype=torch.int32, device=device)


def _check_packed(plan, starts, scale=None):
    q, k, v = plan.q.cpu(), plan.k.cpu(), plan.v.cpu()
    ref, bound = S.packed_attention(q, k, v, starts, scale)
    a, b = starts[0], starts[-1]
    longest = max([0] + [y - x for x, y in zip(starts[:-1], starts[1:])])
    _assert_close(plan.output[a:b], ref[a:b], bound[a:b], longest, v.float().abs().max().item())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_packed_heads(hq, hkv, d, dtype, gpu_device):
    q, k, v, starts, on_gpu = _packed([70, 1, 0, 133, 5], hq, hkv, d, dtype, gpu_device, fused=hq % 3 == 0)
    plan = prepare_packed_gqa(q, k, v, on_gpu)
    _check_packed(plan, starts)
    plan.check_inputs()


@pytest.mark.parametrize("lengths", [[1], [1, 1, 1], [0, 0, 2, 0], [64], [63, 65, 1, 129], [256, 255, 257], [1100, 3],
                                     [31, 32, 33] * 5, [2049], [0, 700, 0]], ids=str)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64)])
def test_packed_lengths(lengths, hq, hkv, d, gpu_device):
    q, k, v, starts, on_gpu = _packed(lengths, hq, hkv, d, torch.bfloat16, gpu_device)
    _check_packed(prepare_packed_gqa(q, k, v, on_gpu), starts)


def test_packed_many_sequences(gpu_device):
    lengths = [(7 * i) % 23 for i in range(700)]
    q, k, v, starts, on_gpu = _packed(lengths, 4, 1, 64, torch.float16, gpu_device, first=3, behind=4)
    _check_packed(prepare_packed_gqa(q, k, v, on_gpu), starts)


@pytest.mark.parametrize("fused", [False, True])
def test_packed_rows_of_no_sequence(fused, gpu_device):
    """Rows before the first and behind the last sequence keep their bits,
    whatever their inputs hold, and reach no other row."""
    q, k, v, starts, on_gpu = _packed([40, 90], 8, 2, 128, torch.bfloat16, gpu_device, fused, first=9, behind=21)
    for t in (q, k, v):
        t[:9], t[139:] = float("nan"), float("inf")
    out = torch.full((160, 8, 128), 7.0, dtype=torch.bfloat16, device=gpu_device)
    plan = prepare_packed_gqa(q, k, v, on_gpu, out)
    assert (out[:9] == 7).all() and (out[139:] == 7).all()
    _check_packed(plan, starts)
    plan.check_inputs()
    on_gpu.fill_(50)          # all sequences empty
    out.fill_(5.0)
    plan.run()
    assert (out == 5).all()


def test_packed_nothing_to_do(gpu_device):
    q, k, v, _, on_gpu = _packed([4], 8, 2, 128, torch.bfloat16, gpu_device)
    assert prepare_packed_gqa(q[:0], k[:0], v[:0], on_gpu[:1]).run().shape == (0, 8, 128)
    plan = prepare_packed_gqa(q, k, v, on_gpu[:1], torch.ones_like(q))
    assert (plan.run() == 1).all()
    plan.check_inputs()


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, torch.bfloat16), (6, 2, 64, torch.float16)])
def test_packed_non_finite(hq, hkv, d, dtype, gpu_device):
    """Keys and values that a token does not see (later tokens, other sequences)
    do not reach it, finite or not; its own do."""
    lengths = [100, 300, 90]
    q, k, v, starts, on_gpu = _packed(lengths, hq, hkv, d, dtype, gpu_device)
    clean = prepare_packed_gqa(q, k, v, on_gpu).output.clone()
    for t, what in ((k, "k"), (v, "v")):
        for row, value in ((250, float("nan")), (250, float("inf")), (399, float("-inf")), (100, float("nan")),
                           (117, float("inf")), (262, torch.finfo(dtype).min)):
            kept = t[row].clone()
            t[row] = value
            plan = prepare_packed_gqa(q, k, v, on_gpu)
            out = plan.output
            t[row] = kept
            assert torch.equal(out[:100], clean[:100]) and torch.equal(out[400:], clean[400:]), (what, row, value)
            before = out[100:row]
            assert torch.isfinite(before).all(), (what, row, value)
            if row > 100:
                ref, bound = S.packed_attention(q.cpu(), k.cpu(), v.cpu(), starts)
                _assert_close(before, ref[100:row], bound[100:row], 300, v.float().abs().max().item())
            if what == "v" and value != torch.finfo(dtype).min:
                assert not torch.isfinite(out[row:400]).any()
            if what == "k" and value != value:
                assert out[row:400].isnan().all()


def test_packed_scale_and_large_scores(gpu_device):
    """An explicit scale, and keys like their token's queries, growing along the
    sequence (the running maximum moves all the time)."""
    q, k, v, starts, on_gpu = _packed([500, 77], 8, 2, 128, torch.bfloat16, gpu_device)
    _check_packed(prepare_packed_gqa(q, k, v, on_gpu, scale=0.02), starts, 0.02)
    k.copy_(q.view(577, 2, 4, 128)[:, :, 0] * (torch.arange(577, device=gpu_device) / 577)[:, None, None])
    out = prepare_packed_gqa(q, k, v, on_gpu).output
    ref, bound = S.packed_attention(q.cpu(), k.cpu(), v.cpu(), starts)
    # A token's own key has sum |q k| = sum q^2, up to 200 where independent rows
    # have 82: its score's rounding counts up to three times.
    tol = S.tolerance(ref, bound, torch.bfloat16, 500, 5.0) + bound * 2.0 ** -11
    assert ((out.double().cpu() - ref).abs() <= tol).all()


def test_packed_replays_and_streams(gpu_device):
    """One captured run on new values and new starts, replayed on another stream
    with eager runs between, gives the eager bits, and every run the same."""
    q, k, v, starts, on_gpu = _packed([300, 0, 45, 600], 32, 8, 128, torch.bfloat16, gpu_device)
    plan, other = prepare_packed_gqa(q, k, v, on_gpu), prepare_packed_gqa(q, k, v, on_gpu)
    side = torch.cuda.Stream(device=gpu_device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan.run()
    for i, lengths in enumerate(([300, 0, 45, 600], [945, 0, 0, 0], [1, 2, 3, 4], [100, 200, 300, 345])):
        on_gpu.copy_(torch.tensor(_starts(lengths), dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        plan.output.zero_()
        other.output.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        replay = plan.output.clone()
        assert torch.equal(replay, other.run())
        assert torch.equal(replay, other.run())
        _check_packed(plan, _starts(lengths))


def test_packed_bad_starts(gpu_device):
    """Starts outside [0, N] or falling are reported and read nothing outside."""
    q, k, v, starts, on_gpu = _packed([40, 90], 8, 2, 128, torch.bfloat16, gpu_device)
    plan = prepare_packed_gqa(q, k, v, on_gpu)
    clean = plan.output.clone()
    plan.check_inputs()
    for bad in ([0, 40, 131], [-3, 40, 130], [0, 40, 20], [0, 2 ** 31 - 1, 130], [-2 ** 31, 40, 130]):
        on_gpu.copy_(torch.tensor(bad, dtype=torch.int32))
        plan.run()
        with pytest.raises(ValueError, match="starts"):
            plan.check_inputs()
        plan.check_inputs()  # reported once
    on_gpu.copy_(torch.tensor(starts, dtype=torch.int32))
    assert torch.equal(plan.run(), clean)


@pytest.mark.parametrize("count", [5, 64, 100, 3000])
def test_packed_starts_without_order(count, gpu_device):
    """Starts in any order are taken as the largest so far within [0, N], found by
    a wave, by the sorted list and by the list of many sequences."""
    n = 400
    q, k, v, _, _ = _packed([n], 4, 2, 64, torch.bfloat16, gpu_device)
    g = torch.Generator().manual_seed(count)
    raw = torch.randint(-200, 700, (count + 1,), generator=g)
    if count > 64:  # most of them within a narrow range, rising slowly
        raw = (torch.arange(count + 1) * n // count + torch.randint(-30, 30, (count + 1,), generator=g))
    raw[0] = 7
    starts = torch.cummax(raw.clamp(0, n), 0).values.tolist()
    out = torch.full((n, 4, 64), 3.0, dtype=torch.bfloat16, device=gpu_device)
    plan = prepare_packed_gqa(q, k, v, raw.to(torch.int32).to(gpu_device), out)
    _check_packed(plan, starts)
    assert (out[:7] == 3).all() and (out[starts[-1]:] == 3).all()
    with pytest.raises(ValueError, match="starts"):
        plan.check_inputs()


@pytest.mark.parametrize("count,hq,hkv,d", [(80, 40, 1, 64), (40, 16, 1, 128), (90, 24, 2, 128)])
def test_packed_few_rounds(count, hq, hkv, d, gpu_device):
    """More tiles than CUs, in a second round of workgroups that is not full."""
    lengths = [(7 * i) % 20 * (5 if count < 64 else 1) for i in range(count)]
    q, k, v, starts, on_gpu = _packed(lengths, hq, hkv, d, torch.bfloat16, gpu_device)
    plan = prepare_packed_gqa(q, k, v, on_gpu)
    _check_packed(plan, starts)
    plan.check_inputs()


@pytest.mark.parametrize("lengths,hq,hkv,d", [
    ([1500, 0, 1100], 32, 8, 128), ([(130 * i) % 700 + 1 for i in range(9)], 32, 8, 128), ([300] * 7, 16, 16, 128),
    ([(37 * i) % 290 for i in range(64)], 12, 4, 64), ([900, 5, 0, 260], 64, 1, 128), ([0, 1024, 1025, 0], 16, 2, 64)])
def test_packed_longest_first(lengths, hq, hkv, d, gpu_device):
    """Up to 64 sequences with somewhat more tiles than CUs, as they are and with rows
    of no sequence around them, every row in some tile exactly once."""
    for first, behind in ((0, 0), (3, 40)):
        q, k, v, starts, on_gpu = _packed(lengths, hq, hkv, d, torch.bfloat16, gpu_device, first=first, behind=behind)
        out = torch.full_like(q, 7.0).contiguous()
        plan = prepare_packed_gqa(q, k, v, on_gpu, out)
        _check_packed(plan, starts)
        assert (out[:first] == 7).all() and (out[starts[-1]:] == 7).all()
        plan.check_inputs()


@pytest.mark.parametrize("count", [2100, 5000])
def test_packed_many_sequences_listed(count, gpu_device):
    """More sequences than the sorting workgroup holds in LDS."""
    lengths = [(5 * i) % 7 for i in range(count)]
    q, k, v, starts, on_gpu = _packed(lengths, 2, 1, 64, torch.bfloat16, gpu_device)
    plan = prepare_packed_gqa(q, k, v, on_gpu)
    _check_packed(plan, starts)
    plan.check_inputs()


# ---- paged decode -----------------------------------------------------------------


def _paged(lengths, hq, hkv, d, page, dtype, device, order="heads", spare=3, seed=0, wide="narrow"):
    """Pages in a shuffled order; the places behind each sequence's end and the
    spare pages hold NaN, table entries behind the last page an impossible one.
    ``wide``: see WIDE; "long" adds a sequence to ``lengths``."""
    if wide == "long":
        lengths.append(1000)
    g = torch.Generator().manual_seed(seed + sum(lengths) + page)
    used = [-(-n // page) for n in lengths]
    count, width = sum(used) + spare, max(used) + 2 if wide == "narrow" else 1000
    perm = torch.randperm(count, generator=g).tolist()
    shape = (count, hkv, page, d) if order == "heads" else (count, page, hkv, d)
    kv = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)]
    if order != "heads":
        kv = [t.transpose(1, 2) for t in kv]
    tables, at = [], 0
    for n, u in zip(lengths, used):
        rows = perm[at:at + u]
        tables.append(rows + [1 << 29] * (width - u))
        if n % page:
            for t in kv:
                t[rows[-1], :, n % page:] = float("nan")
        at += u
    for t in kv:
        t[perm[at:]] = float("nan")
    q = torch.randn(len(lengths), hq, d, generator=g).to(dtype)

    def on_gpu(t):
        if order == "heads":
            return t.to(device)
        return t.transpose(1, 2).contiguous().to(device).transpose(1, 2)

    return (q.to(device), on_gpu(kv[0]), on_gpu(kv[1]), tables,
            torch.tensor(tables, dtype=torch.int32, device=device), torch.tensor(lengths, dtype=torch.int32, device=device))


def _check_paged(plan, tables, lengths, scale=None):
    q, k, v = plan.q.cpu(), plan.k_pages.cpu(), plan.v_pages.cpu()
    ref, bound = S.paged_attention(q, k, v, tables, lengths, scale)
    _assert_close(plan.output, ref, bound, max(lengths), v.float().nan_to_num(0).abs().max().item())
    for b, n in enumerate(lengths):
        if n == 0:
            assert (plan.output[b] == 0).all()


@pytest.mark.parametrize("wide", WIDE)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_paged_heads(hq, hkv, d, dtype, wide, gpu_device):
    lengths = [37, 0, 1, 200, 64]
    q, k, v, tables, gt, gl = _paged(lengths, hq, hkv, d, 16, dtype, gpu_device, wide=wide)
    plan = prepare_paged_gqa(q, k, v, gt, gl)
    _check_paged(plan, tables, lengths)
    plan.check_inputs()


@pytest.mark.parametrize("lengths,page", [
    ([1], 16), ([16], 16), ([17], 16), ([0], 16), ([0, 0, 5], 16), ([31, 32, 33], 16), ([700], 16), ([5000], 32),
    ([1000, 1, 47, 48, 49], 48), ([1500, 3], 1024), ([1024, 1025], 1024), ([9000, 12, 0, 400], 80),
    ([(37 * i) % 150 for i in range(130)], 16)], ids=lambda x: str(x)[:24])
@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("wide", WIDE)
def test_paged_lengths(lengths, page, order, wide, gpu_device):
    lengths = list(lengths)
    q, k, v, tables, gt, gl = _paged(lengths, 8, 2, 128, page, torch.bfloat16, gpu_device, order, wide=wide)
    plan = prepare_paged_gqa(q, k, v, gt, gl)
    _check_paged(plan, tables, lengths)
    plan.check_inputs()


def test_paged_long_fp16_d64(gpu_device):
    lengths = [20000, 3000, 1]
    q, k, v, tables, gt, gl = _paged(lengths, 14, 2, 64, 64, torch.float16, gpu_device)
    _check_paged(prepare_paged_gqa(q, k, v, gt, gl, scale=0.25), tables, lengths, 0.25)


@pytest.mark.parametrize("wide", WIDE)
def test_paged_many_rows(wide, gpu_device):
    """More sequences than a wave has lanes several times over, most of them empty."""
    lengths = [0 if i % 3 else (i * 7) % 60 for i in range(1500)]
    q, k, v, tables, gt, gl = _paged(lengths, 4, 2, 64, 16, torch.bfloat16, gpu_device, wide=wide)
    _check_paged(prepare_paged_gqa(q, k, v, gt, gl), tables, lengths)


def test_paged_shared_pages_and_strided_tables(gpu_device):
    """Sequences that share pages, tables and q as views of wider tensors, and
    keys and values interleaved in one allocation."""
    page, hkv, d = 16, 2, 128
    both = torch.randn(20, 2, hkv, page, d).to(torch.bfloat16).to(gpu_device)
    k, v = both[:, 0], both[:, 1]
    wide = torch.full((4, 40), -1, dtype=torch.int32, device=gpu_device)
    tables = [[3, 4, 5, 0], [3, 4, 6, 0], [3, 9, 9, 9], [19, 0, 0, 0]]
    wide[:, 8:12] = torch.tensor(tables, dtype=torch.int32)
    q = torch.randn(4, 24, d).to(torch.bfloat16).to(gpu_device)[:, 3:11]
    lengths = [45, 40, 64, 16]
    gl = torch.tensor(lengths, dtype=torch.int32, device=gpu_device)
    plan = prepare_paged_gqa(q, k, v, wide[:, 8:12], gl)
    _check_paged(plan, tables, lengths)
    plan.check_inputs()


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (14, 2, 64), (40, 2, 128)])
def test_paged_many_sequences(hq, hkv, d, gpu_device):
    """Enough sequences that they are not all worked on at once."""
    lengths = [(97 * i) % 400 for i in range(40960 // (hkv * d))]
    q, k, v, tables, gt, gl = _paged(lengths, hq, hkv, d, 16, torch.bfloat16, gpu_device)
    plan = prepare_paged_gqa(q, k, v, gt, gl)
    _check_paged(plan, tables, lengths)
    plan.check_inputs()


@pytest.mark.parametrize("wide", WIDE)
def test_paged_non_finite(wide, gpu_device):
    """Values that are seen and not finite reach the output, as do NaN keys; a key
    of -inf score drops out; other sequences keep their bits."""
    lengths = [300, 300, 300, 300]
    q, k, v, tables, gt, gl = _paged(lengths, 8, 2, 128, 16, torch.bfloat16, gpu_device, wide=wide)
    plan = prepare_paged_gqa(q, k, v, gt, gl)
    clean = plan.output.clone()
    v[tables[0][7], 0, 3, 100] = float("inf")
    k[tables[1][18], 1, 11, 5] = float("nan")          # the last keys of row 1
    sign = float(q[2, 1, 9] > 0) * 2 - 1
    k[tables[2][0], 0, 0, 9] = -float("inf") * sign    # -inf or +inf score by the head's sign
    out = plan.run()
    assert torch.equal(out[3], clean[3]) and torch.equal(out[0, 4:], clean[0, 4:]) and torch.equal(out[2, 4:], clean[2, 4:])
    assert (out[0, :4, 100] == float("inf")).all() and torch.isfinite(out[0, :4, :100]).all()
    assert out[1, 4:].isnan().all() and torch.equal(out[1, :4], clean[1, :4])
    for h in range(4):
        if (q[2, h, 9] > 0) == (sign > 0):
            assert torch.isfinite(out[2, h]).all()
        else:
            assert out[2, h].isnan().all()


@pytest.mark.parametrize("wide", WIDE)
def test_paged_bad_pages_and_lengths(wide, gpu_device):
    """Page numbers outside the cache are left out, lengths outside the table taken
    as the nearest within; both are reported, the other sequences unchanged."""
    lengths = [60, 33, 100]
    q, k, v, tables, gt, gl = _paged(lengths, 8, 2, 128, 16, torch.bfloat16, gpu_device, wide=wide)
    plan = prepare_paged_gqa(q, k, v, gt, gl)
    clean = plan.output.clone()
    plan.check_inputs()
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        gt[0, 1] = bad
        out = plan.run()
        assert torch.equal(out[1:], clean[1:])
        assert plan.read_status() == N.GQA_STATUS_BAD_PAGE and plan.read_status() == 0
        keys = [(tables[0][j // 16], j % 16) for j in range(60) if j // 16 != 1]
        rows = torch.tensor([p for p, _ in keys]), torch.tensor([r for _, r in keys])
        ref, bound = S.attention_rows(q[0].cpu(), k.cpu()[rows[0], :, rows[1]], v.cpu()[rows[0], :, rows[1]])
        _assert_close(out[0], ref, bound, 60, 5.0)
    gt[0, 1] = tables[0][1]
    gt[1] = -1                                   # a sequence without any page
    assert (plan.run()[1] == 0).all() and plan.read_status() == N.GQA_STATUS_BAD_PAGE
    gt[1] = torch.tensor(tables[1], dtype=torch.int32)
    gl[1] = -4
    ref, bound = S.paged_attention(q.cpu(), k.cpu(), v.cpu(), tables, lengths)
    out = plan.run()
    assert (out[1] == 0).all()
    _assert_close(out[::2], ref[::2], bound[::2], 100, 5.0)
    assert plan.read_status() == N.GQA_STATUS_BAD_BOUNDS
    gl[1] = 2 ** 31 - 1
    out = plan.run()
    _assert_close(out[::2], ref[::2], bound[::2], 100, 5.0)
    assert plan.read_status() == N.GQA_STATUS_BAD_BOUNDS | N.GQA_STATUS_BAD_PAGE


def test_paged_offsets_past_32_bits(gpu_device):
    """Pages more than 2^32 bytes from the base, of heads and of tokens outermost."""
    count, hkv, page, d = 20000, 8, 128, 128
    for order in ("heads", "tokens"):
        shape = (count, hkv, page, d) if order == "heads" else (count, page, hkv, d)
        k, v = (torch.empty(shape, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
        assert k.numel() * 2 > 1 << 32
        tables = [[count - 1, 0, count // 2, count - 2], [count - 3, count - 5, 17, 1]]
        for p in sum(tables, []):
            k[p].normal_()
            v[p].normal_()
        kk, vv = (k, v) if order == "heads" else (k.transpose(1, 2), v.transpose(1, 2))
        q = torch.randn(2, 32, d).to(torch.bfloat16).to(gpu_device)
        lengths = [500, 385]
        plan = prepare_paged_gqa(q, kk, vv, torch.tensor(tables, dtype=torch.int32, device=gpu_device),
                                 torch.tensor(lengths, dtype=torch.int32, device=gpu_device))
        rows = sorted(set(sum(tables, [])))
        small = [[rows.index(p) for p in t] for t in tables]
        ref, bound = S.paged_attention(q.cpu(), kk[rows].cpu(), vv[rows].cpu(), small, lengths)
        _assert_close(plan.output, ref, bound, 500, 6.0)
        del plan, k, v, kk, vv


@pytest.mark.parametrize("wide", WIDE)
def test_paged_replays_and_streams(wide, gpu_device):
    """One captured run, replayed on another stream while lengths, tables and
    values change, gives the eager bits; runs repeat their bits."""
    lengths = [1500, 1, 0, 333]
    q, k, v, tables, gt, gl = _paged(lengths, 32, 8, 128, 16, torch.bfloat16, gpu_device, wide=wide)
    k.nan_to_num_(0.5)
    v.nan_to_num_(0.5)
    plan, other = prepare_paged_gqa(q, k, v, gt, gl), prepare_paged_gqa(q, k, v, gt, gl)
    side = torch.cuda.Stream(device=gpu_device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan.run()
    for i, now in enumerate(([1500, 1, 0, 333], [3, 1, 0, 1], [0, 0, 0, 0], [1488, 16, 0, 320], [1, 0, 0, 336])):
        now = now + lengths[4:]
        gl.copy_(torch.tensor(now, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        replay = plan.output.clone()
        assert torch.equal(replay, other.run())
        assert torch.equal(replay, other.run())
        _check_paged(plan, tables, now)


# ---- all of them together ----------------------------------------------------------


def test_serving_a_batch(gpu_device):
    """Prompts, decode steps from a captured graph, forks, frees and a compaction:
    every layer's attention equals dense attention over each row's own history."""
    layers, hq, hkv, d, rows = 2, 8, 2, 64, 6
    c = PagedKVCache(80, 16, hkv, d, sequences=rows, max_pages=12, max_tokens=256, layers=layers, device=gpu_device)
    history = [[[] for _ in range(rows)] for _ in range(layers)]  # (k, v) per token
    g = torch.Generator().manual_seed(1)

    def rnd(n):
        return torch.randn(n, hq + 2 * hkv, d, generator=g).to(torch.bfloat16).to(gpu_device).split([hq, hkv, hkv], 1)

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device=gpu_device)

    def check(out, q, layer, row, upto=None):
        ks, vs = (torch.stack([t[i] for t in history[layer][row][:upto]]) for i in (0, 1))
        ref, bound = S.attention_rows(q.cpu(), ks, vs)
        _assert_close(out, ref, bound, len(ks), 6.0)

    def prompts(counts):
        c.reserve(i32(counts))
        starts = _starts(counts)
        for layer in range(layers):
            q, k, v = rnd(starts[-1])
            c.append(layer, k, v)
            out = prepare_packed_gqa(q, k, v, c.starts).output
            for r, n in enumerate(counts):
                for i in range(n):
                    history[layer][r].append((k[starts[r] + i].cpu(), v[starts[r] + i].cpu()))
                    if i % 13 == 0 or i == n - 1:
                        check(out[starts[r] + i], q[starts[r] + i], layer, r, i + 1)

    prompts([40, 0, 77, 0, 5, 0])
    counts = i32([0] * rows)
    qkv = [rnd(rows) for _ in range(layers)]
    plans = [prepare_paged_gqa(qkv[i][0], c.k[i], c.v[i], c.tables, c.lengths) for i in range(layers)]
    torch.cuda.synchronize()
    step = torch.cuda.CUDAGraph()
    with torch.cuda.graph(step):
        c.reserve(counts, stride=1)
        for layer in range(layers):
            c.append(layer, qkv[layer][1], qkv[layer][2])
            plans[layer].run()

    def decode(active):
        counts.copy_(i32(active))
        for layer in range(layers):
            for t, new in zip(qkv[layer], rnd(rows)):
                t.copy_(new)
        step.replay()
        for layer in range(layers):
            for r in range(rows):
                if active[r]:
                    history[layer][r].append((qkv[layer][1][r].cpu(), qkv[layer][2][r].cpu()))
                if history[layer][r]:
                    check(plans[layer].output[r], qkv[layer][0][r], layer, r)
                else:
                    assert (plans[layer].output[r] == 0).all()

    for _ in range(4):
        decode([1, 0, 1, 0, 1, 0])
    c.fork(i32([0, 2]), i32([1, 3]))
    for layer in range(layers):
        history[layer][1], history[layer][3] = list(history[layer][0]), list(history[layer][2])
    for i in range(5):
        decode([1, 1, i % 2, 1, 1, 0])
    c.free(i32([2, 4]))
    for layer in range(layers):
        history[layer][2], history[layer][4] = [], []
    c.compact()
    decode([1, 1, 0, 0, 0, 0])
    prompts([0, 0, 30, 0, 0, 61])
    for _ in range(3):
        decode([1] * 4 + [0, 1])
    assert c.read_status() == 0
    for p in plans:
        p.check_inputs()


def test_packed_offsets_past_32_bits(gpu_device):
    """Token strides that put the last keys, values and queries more than 2^32
    bytes from the base."""
    n, wide = 70000, 1 << 16
    base = torch.empty(n, wide, dtype=torch.bfloat16, device=gpu_device)
    assert base.numel() * 2 > 1 << 33
    g = torch.Generator(device=gpu_device).manual_seed(5)
    q, k, v = (base[:, i * 4096:i * 4096 + h * 64].unflatten(1, (h, 64)) for i, h in enumerate((8, 1, 1)))
    for t in (q, k, v):
        t.copy_(torch.randn(t.shape, generator=g, device=gpu_device))
    starts = [0, 69300, 69301, 70000]
    plan = prepare_packed_gqa(q, k, v, torch.tensor(starts, dtype=torch.int32, device=gpu_device))
    qc, kc, vc = q.cpu(), k.cpu(), v.cpu()
    for t in (0, 31, 4097, 32768, 69299, 69300, 69301, 69999):
        first = max(s for s in starts[:-1] if s <= t)
        ref, bound = S.attention_rows(qc[t], kc[first:t + 1], vc[first:t + 1])
        _assert_close(plan.output[t], ref, bound, t + 1 - first, 6.0)
    plan.check_inputs()


def test_paged_as_many_rows_as_allowed(gpu_device):
    """2^16 sequences of 0 to 3 pages that share 50 pages."""
    b, pages = 1 << 16, 50
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(pages, 1, 16, 64, generator=g).to(torch.float16).to(gpu_device) for _ in range(2))
    tables = torch.randint(0, pages, (b, 3), generator=g, dtype=torch.int32)
    lengths = torch.randint(0, 49, (b,), generator=g, dtype=torch.int32)
    q = torch.randn(b, 2, 64, generator=g).to(torch.float16)
    plan = prepare_paged_gqa(q.to(gpu_device), k, v, tables.to(gpu_device), lengths.to(gpu_device))
    rows = list(range(0, b, 997)) + [b - 1]
    ref, bound = S.paged_attention(q[rows], k.cpu(), v.cpu(), tables[rows].tolist(), lengths[rows].tolist())
    _assert_close(plan.output[rows], ref, bound, 48, 5.0)
    assert (plan.output[(lengths == 0).to(gpu_device)] == 0).all()
    plan.check_inputs()


def test_two_plans_on_two_streams(gpu_device):
    """Plans of their own run side by side, with the same inputs and pages."""
    q, k, v, starts, on_gpu = _packed([900, 3, 400], 16, 4, 128, torch.bfloat16, gpu_device)
    pq, pk, pv, tables, gt, gl = _paged([2000, 5, 700], 16, 4, 128, 16, torch.bfloat16, gpu_device)
    packed = [prepare_packed_gqa(q, k, v, on_gpu) for _ in range(2)]
    paged = [prepare_paged_gqa(pq, pk, pv, gt, gl) for _ in range(2)]
    want = packed[0].output.clone(), paged[0].output.clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=gpu_device) for _ in range(2)]
    for _ in range(3):
        for p in packed + paged:
            p.output.zero_()
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for _ in range(4):
                    (packed if i else paged)[i].run()
                    (paged if i else packed)[i].run()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(packed[i].output, want[0]) and torch.equal(paged[i].output, want[1])
