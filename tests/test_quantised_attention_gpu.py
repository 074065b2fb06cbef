"""Decode attention over a microscaled cache against attention in 64 bits over what its
elements stand for (MI355X only).  Those values are numbers of q's type, so that the
tolerances are those of the 16-bit cache: oracle/serving_oracle.py, tolerance()."""
import pytest
import torch

from llm_gpu_kernels_amd import PagedKVCache, _native as N, prepare_paged_gqa, prepare_qk_norm_rope
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu

HEADS = [(32, 8, 128), (8, 8, 128), (12, 4, 64), (14, 2, 64), (6, 6, 64), (16, 1, 128), (40, 2, 128), (64, 1, 64)]
TYPES = [torch.bfloat16, torch.float16]
STORAGES = ["mxfp8", "mxfp4"]
ELEMENTS = {"mxfp8": torch.float8_e4m3fn, "mxfp4": torch.float4_e2m1fn_x2}
WIDE = ["narrow", "wide", "long"]  # as in the tests of the 16-bit cache: three ways of sharing out the work


def _assert_close(out, ref, bound, keys, vmax):
    off = (out.double().cpu() - ref).abs()
    tol = S.tolerance(ref, bound, out.dtype, keys, vmax)
    assert torch.isfinite(out).all()
    worst = (off / tol.clamp(min=1e-30)).max().item()
    assert worst <= 1.0, worst


class Pages:
    """Quantised N(0, 1) rows in pages without order; places behind each sequence's end
    and spare pages hold NaN (scale 255 and, of eight bits, NaN elements), table entries
    behind the last page an impossible number."""

    def __init__(self, lengths, hq, hkv, d, page, dtype, storage, device, spare=3, wide="narrow", swapped=False):
        if wide == "long":
            lengths.append(1000)
        g = torch.Generator().manual_seed(sum(lengths) + page + hq)
        used = [-(-n // page) for n in lengths]
        count, width = sum(used) + spare, max(used) + 2 if wide == "narrow" else 1000
        perm = torch.randperm(count, generator=g).tolist()
        self.lengths, self.tables, at = lengths, [], 0
        absent = torch.ones(count, page, dtype=torch.bool)
        for n, u in zip(lengths, used):
            rows = perm[at:at + u]
            self.tables.append(rows + [1 << 29] * (width - u))
            for i, p in enumerate(rows):
                absent[p, :n - i * page] = False
            at += u
        self.values, self.gpu = [], []
        for _ in range(2):
            x = torch.randn(count, hkv, page, d, generator=g).to(dtype)
            codes, scales = S.mx_quantise(x, storage, dtype)
            self.values.append(S.mx_values(codes, scales, storage))
            held = S.mx_pack(codes, storage)
            held = torch.where(absent[:, None, :, None], torch.tensor(255, dtype=torch.uint8), held)
            scales = torch.where(absent[:, None, :, None], torch.tensor(255, dtype=torch.uint8), scales).transpose(2, 3)
            for t, kind in ((held, ELEMENTS[storage]), (scales, torch.float8_e8m0fnu)):
                if swapped:  # heads outermost, then pages
                    t = t.transpose(0, 1).contiguous().to(device).transpose(0, 1)
                self.gpu.append(t.contiguous().to(device).view(kind) if not swapped else t.view(kind))
        self.q = torch.randn(len(lengths), hq, d, generator=g).to(dtype).to(device)
        self.gt = torch.tensor(self.tables, dtype=torch.int32, device=device)
        self.gl = torch.tensor(lengths, dtype=torch.int32, device=device)

    def plan(self, **kw):
        k, ks, v, vs = self.gpu
        return prepare_paged_gqa(self.q, k, v, self.gt, self.gl, k_scales=ks, v_scales=vs, **kw)

    def reference(self, scale=None, rows=slice(None)):
        k, v = self.values
        return S.paged_attention(self.q.cpu()[rows], k, v, self.tables[rows], self.lengths[rows], scale)

    def check(self, plan, scale=None):
        ref, bound = self.reference(scale)
        _assert_close(plan.output, ref, bound, max(self.lengths), self.values[1].abs().max().item())
        for b, n in enumerate(self.lengths):
            if n == 0:
                assert (plan.output[b] == 0).all()
        plan.check_inputs()


@pytest.mark.parametrize("wide", WIDE)
@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_heads(hq, hkv, d, dtype, storage, wide, gpu_device):
    p = Pages([37, 0, 1, 200, 64], hq, hkv, d, 16, dtype, storage, gpu_device, wide=wide)
    p.check(p.plan())


@pytest.mark.parametrize("lengths,page", [
    ([1], 16), ([16], 16), ([17], 16), ([0], 16), ([0, 0, 5], 16), ([31, 32, 33], 16), ([700], 16), ([5000], 32),
    ([1000, 1, 47, 48, 49], 48), ([1500, 3], 1024), ([1024, 1025], 1024), ([9000, 12, 0, 400], 80),
    ([(37 * i) % 150 for i in range(130)], 16)], ids=lambda x: str(x)[:24])
@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("wide", WIDE)
def test_lengths(lengths, page, storage, wide, gpu_device):
    p = Pages(list(lengths), 8, 2, 128, page, torch.bfloat16, storage, gpu_device, wide=wide, swapped=page == 48)
    p.check(p.plan())


@pytest.mark.parametrize("storage", STORAGES)
def test_long_fp16_d64(storage, gpu_device):
    p = Pages([20000, 3000, 1], 14, 2, 64, 64, torch.float16, storage, gpu_device)
    p.check(p.plan(scale=0.25), 0.25)


@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("wide", WIDE)
def test_many_rows(storage, wide, gpu_device):
    """More sequences than a wave has lanes several times over, most of them empty."""
    p = Pages([0 if i % 3 else (i * 7) % 60 for i in range(1500)], 4, 2, 64, 16, torch.bfloat16, storage, gpu_device, wide=wide)
    p.check(p.plan())


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (40, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("storage", STORAGES)
def test_many_sequences(hq, hkv, d, storage, gpu_device):
    """Enough sequences that they are not all worked on at once."""
    p = Pages([(97 * i) % 400 for i in range(40960 // (hkv * d))], hq, hkv, d, 16, torch.bfloat16, storage, gpu_device)
    p.check(p.plan())


@pytest.mark.parametrize("wide", WIDE)
@pytest.mark.parametrize("storage", STORAGES)
def test_not_finite(storage, wide, gpu_device):
    """A block that is NaN reaches the heads that see it, no others."""
    p = Pages([300, 300, 300], 8, 2, 128, 16, torch.bfloat16, storage, gpu_device, wide=wide)
    plan = p.plan()
    clean = plan.output.clone()
    _, ks, _, vs = p.gpu
    vs.view(torch.uint8)[p.tables[0][7], 0, 3, 3] = 255   # dims 96 to 127 of a value
    ks.view(torch.uint8)[p.tables[1][18], 1, 0, 11] = 255  # the last keys of row 1
    out = plan.run()
    assert torch.equal(out[2:], clean[2:]) and torch.equal(out[0, 4:], clean[0, 4:])
    assert out[0, :4, 96:].isnan().all() and torch.equal(out[0, :4, :96], clean[0, :4, :96])
    assert out[1, 4:].isnan().all() and torch.equal(out[1, :4], clean[1, :4])


@pytest.mark.parametrize("wide", WIDE)
@pytest.mark.parametrize("storage", STORAGES)
def test_bad_pages_and_lengths(storage, wide, gpu_device):
    p = Pages([60, 33, 100], 8, 2, 128, 16, torch.bfloat16, storage, gpu_device, wide=wide)
    plan = p.plan()
    clean = plan.output.clone()
    plan.check_inputs()
    for bad in (-1, p.gpu[0].shape[0], 2 ** 31 - 1, -2 ** 31):
        p.gt[0, 1] = bad
        out = plan.run()
        assert torch.equal(out[1:], clean[1:])
        assert plan.read_status() == N.GQA_STATUS_BAD_PAGE and plan.read_status() == 0
        keys = [(p.tables[0][j // 16], j % 16) for j in range(60) if j // 16 != 1]
        rows = torch.tensor([x for x, _ in keys]), torch.tensor([x for _, x in keys])
        ref, bound = S.attention_rows(p.q[0].cpu(), *(t[rows[0], :, rows[1]] for t in p.values))
        _assert_close(out[0], ref, bound, 60, 6.0)
    p.gt[0, 1] = p.tables[0][1]
    p.gt[1] = -1
    assert (plan.run()[1] == 0).all() and plan.read_status() == N.GQA_STATUS_BAD_PAGE
    p.gl[1] = -4
    out = plan.run()
    assert (out[1] == 0).all() and torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    assert plan.read_status() == N.GQA_STATUS_BAD_BOUNDS


@pytest.mark.parametrize("storage", STORAGES)
def test_scales_of_every_size(storage, gpu_device):
    """Values from 2^-100 to 2^100 in one cache: the large ones win where they are seen."""
    p = Pages([50, 50], 4, 2, 64, 16, torch.bfloat16, storage, gpu_device)
    vs, v = p.gpu[3], p.values[1]
    for b, e in ((0, -100), (1, 100)):
        for page in p.tables[b][:4]:
            vs.view(torch.uint8)[page] += e % 256  # (bytes: -100 wraps to what it subtracts)
            v[page] *= 2.0 ** e
    ref, bound = p.reference()
    out = p.plan().output
    for b, e in ((0, -100), (1, 100)):  # the same sums, as powers of two go through every step
        _assert_close((out[b].double() * 2.0 ** -e).to(torch.bfloat16), ref[b] * 2.0 ** -e, bound[b] * 2.0 ** -e, 50, 6.0)


@pytest.mark.parametrize("storage", STORAGES)
def test_offsets_past_32_bits(storage, gpu_device):
    page, hkv, d = 1024, 8, 128
    row = d if storage == "mxfp8" else d // 2
    count = (1 << 32) // (hkv * page * row) + 9
    p = Pages([3 * page - 5, 2 * page + 7], 16, hkv, d, page, torch.float16, storage, gpu_device, spare=0)
    used = p.gpu[0].shape[0]
    big, at = [], [count - 1, 2, count - 3, count // 2, count - 2, count - 5][:used]
    for t in p.gpu:
        x = torch.empty((count,) + t.shape[1:], dtype=torch.uint8, device=gpu_device)
        for i, to in enumerate(at):
            x[to] = t.view(torch.uint8)[i]
        big.append(x.view(t.dtype))
    tables = [[at[x] if x < used else x for x in row] for row in p.tables]
    plan = prepare_paged_gqa(p.q, big[0], big[2], torch.tensor(tables, dtype=torch.int32, device=gpu_device), p.gl,
                             k_scales=big[1], v_scales=big[3])
    p.check(plan)


def test_most_sequences_and_heads(gpu_device):
    """As many as a call allows, 2^16 of each: the last ones are attended too."""
    p = Pages([20], 1, 1, 64, 16, torch.bfloat16, "mxfp4", gpu_device)
    k, ks, v, vs = p.gpu
    many, rows = 2 ** 16, [0, 1, 30000, 2 ** 16 - 1]
    lengths = torch.zeros(many, dtype=torch.int32, device=gpu_device)
    lengths[rows] = 20
    plan = prepare_paged_gqa(p.q.expand(many, 1, 64).contiguous(), k, v, p.gt.expand(many, -1).contiguous(), lengths, k_scales=ks,
                             v_scales=vs)
    plan.check_inputs()
    ref, bound = p.reference()
    for row in rows:
        _assert_close(plan.output[row:row + 1], ref, bound, 20, 6.0)
    plan.output[rows] = 0
    assert (plan.output == 0).all()
    k, ks, v, vs = (t.view(torch.uint8)[p.tables[0][0]][None].expand(1, many, -1, -1).contiguous().view(t.dtype) for t in p.gpu)
    plan = prepare_paged_gqa(p.q.expand(1, many, 64).contiguous(), k, v, torch.zeros_like(p.gt[:, :1]), torch.full_like(p.gl, 16),
                             k_scales=ks, v_scales=vs)
    plan.check_inputs()
    ref, bound = S.paged_attention(p.q.cpu(), *p.values, [p.tables[0][:1]], [16])
    _assert_close(plan.output[:, -1:], ref, bound, 16, 6.0)
    assert (plan.output == plan.output[:, :1]).all()


@pytest.mark.parametrize("storage", STORAGES)
def test_keys_up_to_2_31(storage, gpu_device):
    """The longest sequence that a call allows, of one page over and over: attention over its 16
    keys.  2048 waves take its 2^27 blocks, two at a time, so a sum of a wave has 2^15 terms and
    is off by 2^15 * 2^-24 of its magnitudes at most: the denominator by 2^-9 of itself, O by 2^-9
    of the bound, and the join of 1024 pieces by 2^-13 of both."""
    p = Pages([16], 1, 1, 64, 16, torch.bfloat16, storage, gpu_device)
    k, ks, v, vs = p.gpu
    pages = 2 ** 27 - 1
    tables = torch.full((1, pages), p.tables[0][0], dtype=torch.int32, device=gpu_device)
    lengths = torch.tensor([16 * pages], dtype=torch.int32, device=gpu_device)
    plan = prepare_paged_gqa(p.q, k, v, tables, lengths, k_scales=ks, v_scales=vs)
    plan.check_inputs()
    ref, bound = p.reference()
    off, tol = (plan.output.double().cpu() - ref).abs(), S.tolerance(ref, bound, torch.bfloat16, 16, 6.0)
    assert (off <= tol + bound * (2.0 ** -8 + 2.0 ** -12)).all()


@pytest.mark.parametrize("storage", STORAGES)
def test_two_streams_and_a_graph(storage, gpu_device):
    """Two plans at once on streams of their own, one of them captured and replayed."""
    a = Pages([700, 33, 2000], 8, 2, 128, 16, torch.bfloat16, storage, gpu_device)
    b = Pages([90, 1500], 8, 2, 128, 16, torch.bfloat16, storage, gpu_device, wide="wide")
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
    a.lengths[0] = 650  # the graph reads lengths when it is replayed
    a.gl[0] = 650
    graph.replay()
    torch.cuda.synchronize()
    a.check(pa)


def test_refusals(gpu_device):
    p = Pages([40, 3], 8, 2, 128, 16, torch.bfloat16, "mxfp8", gpu_device)
    k, ks, v, vs = p.gpu
    four = Pages([40, 3], 8, 2, 128, 16, torch.bfloat16, "mxfp4", gpu_device).gpu

    def refused(kind, k=k, v=v, ks=ks, vs=vs, **kw):
        with pytest.raises(kind):
            prepare_paged_gqa(p.q, k, v, p.gt, p.gl, k_scales=ks, v_scales=vs, **kw)

    refused(TypeError, ks=None, vs=None)
    refused(TypeError, vs=None)
    refused(TypeError, ks=ks.view(torch.uint8))
    refused(TypeError, k=k.view(torch.uint8))
    refused(TypeError, v=four[2])
    refused(TypeError, k=p.q, v=p.q)
    refused(ValueError, k=four[0].view(torch.float8_e4m3fn), v=four[2].view(torch.float8_e4m3fn))
    refused(ValueError, ks=ks[:, :1])
    refused(ValueError, vs=vs[:-1])
    refused(ValueError, k=k.transpose(1, 2), v=v.transpose(1, 2))
    tokens_first = k.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(k.dtype)
    refused(ValueError, k=tokens_first)
    refused(ValueError, ks=ks.view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3).view(ks.dtype))
    refused(ValueError, ks=ks.cpu())
    refused(ValueError, out=p.q)


@pytest.mark.parametrize("storage", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, torch.bfloat16), (12, 4, 64, torch.float16)])
def test_serving_steps(hq, hkv, d, dtype, storage, gpu_device):
    """A server's steps: prompts normed, rotated and cached, samples forked, tokens added
    one by one with decode attention, and the history read back."""
    g = torch.Generator().manual_seed(d)
    counts, layers, page = [40, 0, 77, 16], 2, 16
    c = PagedKVCache(60, page, hkv, d, sequences=6, max_pages=12, max_tokens=160, layers=layers, dtype=dtype,
                     storage=storage, device=gpu_device)
    inv_freq = torch.tensor([1e4 ** (-i / (d // 2)) for i in range(d // 2)], device=gpu_device)
    w = [(1 + 0.1 * torch.randn(d, generator=g)).to(dtype).to(gpu_device) for _ in range(2)]
    history = [[([], []) for _ in range(6)] for _ in range(layers)]  # exact keys and values, by row

    def write(n, rows_of_tokens, positions, layer):
        x = torch.randn(n, hq + 2 * hkv, d, generator=g).to(dtype).to(gpu_device)
        q, k, v = x.split([hq, hkv, hkv], dim=1)
        pos = torch.tensor(positions, dtype=torch.int32, device=gpu_device)
        plan = prepare_qk_norm_rope(q, k, pos, inv_freq, *w, v=v, cache=c, layer=layer)
        keys, _ = S.norm_rope(k.cpu(), pos.cpu(), inv_freq.cpu(), w[1].cpu())
        for i, row in enumerate(rows_of_tokens):
            if row >= 0:
                history[layer][row][0].append(keys[i])
                history[layer][row][1].append(v[i].cpu().double())
        return plan

    def held(layer, row, lengths):
        """What the cache stands for, read back, near what was written."""
        n = lengths[row]
        ko, vo = (torch.zeros(n, hkv, d, dtype=dtype, device=gpu_device) for _ in range(2))
        c.gather(layer, torch.tensor([row], dtype=torch.int32, device=gpu_device),
                 torch.tensor([0, n], dtype=torch.int32, device=gpu_device), ko, vo)
        u = {None: torch.finfo(dtype).eps / 2, "mxfp8": 2.0 ** -4, "mxfp4": 2.0 ** -2}[storage]
        for out, exact in zip((ko, vo), history[layer][row]):
            exact = torch.stack(exact)
            top = exact.abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
            # half a step of an element, or of the smallest one under its block's scale
            tol = torch.maximum(u * exact.abs(), {None: 0.0, "mxfp8": 2.0 ** -17, "mxfp4": 2.0 ** -3}[storage] * top)
            assert ((out.cpu().double() - exact).abs() <= tol + 2.0 ** -16).all()
        return ko, vo

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)  # noqa: E731
    c.reserve(i32(counts + [0, 0]))
    rows = [s for s, n in enumerate(counts) for _ in range(n)]
    for layer in range(layers):
        write(len(rows), rows, [i for n in counts for i in range(n)], layer)
    c.fork(i32([2, 0]), i32([4, 5]))
    for layer in range(layers):
        for a, b in ((2, 4), (0, 5)):
            history[layer][b] = (list(history[layer][a][0]), list(history[layer][a][1]))
    lengths = counts + [counts[2], counts[0]]
    for step in range(20):
        grow = [int(n > 0 and (step + s) % 5 > 0) for s, n in enumerate(lengths)]
        c.reserve(i32(grow), stride=1)
        positions = list(lengths)
        lengths = [n + x for n, x in zip(lengths, grow)]
        for layer in range(layers):
            plan = write(6, [s if x else -1 for s, x in enumerate(grow)], positions, layer)
            scales = {} if storage is None else dict(k_scales=c.k_scales[layer], v_scales=c.v_scales[layer])
            att = prepare_paged_gqa(plan.q_out, c.k[layer], c.v[layer], c.tables, c.lengths, **scales)
            if step % 7 == 6:
                for row, n in enumerate(lengths):
                    if n:
                        ko, vo = held(layer, row, lengths)
                        ref, bound = S.attention_rows(plan.q_out[row].cpu(), ko.cpu(), vo.cpu())
                        _assert_close(att.output[row], ref, bound, n, vo.float().abs().max().item())
                    else:
                        assert (att.output[row] == 0).all()
            att.check_inputs()
    c.compact()
    held(1, 4, lengths)
    c.check_inputs()


@pytest.mark.parametrize("wide", WIDE)
@pytest.mark.parametrize("storage", STORAGES)
def test_elements_between_the_smallest_fp16_numbers(storage, wide, gpu_device):
    """Keys and values that fp16 does not hold: attention over them to nearest even.  Large
    queries give scores as of N(0, 1) rows; an output below 2^-14 is off by 2^-25 instead of
    by half a step of its own."""
    p = Pages([300, 77, 1], 8, 2, 128, 16, torch.float16, storage, gpu_device, wide=wide)
    down = 20 if storage == "mxfp8" else 24  # powers of two
    lost = 0
    for i in (0, 1):
        s = p.gpu[2 * i + 1].view(torch.uint8)
        s.copy_(torch.where(s == 255, s, s - down))
        x = p.values[i] * 2.0 ** -down
        p.values[i] = x.half().double()
        lost += int((p.values[i] != x).sum())
    assert lost > 0
    p.q *= 2.0 ** 12
    scale = 128 ** -0.5 * 2.0 ** (down - 12)
    plan = p.plan(scale=scale)
    ref, bound = p.reference(scale)
    tol = S.tolerance(ref, bound, torch.float16, max(p.lengths), p.values[1].abs().max().item()) + 2.0 ** -25
    assert ((plan.output.double().cpu() - ref).abs() <= tol).all()
    plan.check_inputs()
