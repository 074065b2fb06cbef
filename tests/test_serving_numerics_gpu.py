"""Packed and paged attention where the numbers are extreme: probabilities far
below the largest, scores of millions (MI355X only).  References in 64 bits and
tolerances as in oracle/serving_oracle.py, tolerance()."""
import pytest
import torch

from llm_gpu_kernels_amd import _native as N, prepare_packed_gqa, prepare_paged_gqa
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def _assert_rows(out, q, k, v, keys_of_row, rows, scale=None):
    """Rows ``rows`` of ``out`` [rows, Hq, D]; row r sees its first
    keys_of_row(r) keys of k, v [n, Hkv, D].  tolerance() takes the outputs'
    rounding as relative; fp16 ones below 2^-14 are multiples of 2^-24, so off by
    2^-25."""
    step = 2.0 ** -25 if out.dtype == torch.float16 else 1e-30
    vmax = v.float().abs().max().item()
    for r in rows:
        n = keys_of_row(r)
        ref, bound = S.attention_rows(q[r].cpu(), k[:n].cpu(), v[:n].cpu(), scale)
        off = (out[r].double().cpu() - ref).abs()
        worst = (off / (S.tolerance(ref, bound, out.dtype, n, vmax) + step)).max().item()
        assert worst <= 1.0, (r, worst)


def _sink(n, rows, hq, hkv, d, nats, dtype, seed):
    """Keys of scores around 0, and a first one with a value of 0 that lies
    ``nats`` above them for every query."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(s, generator=g) for s in ((rows, hq, d), (n, hkv, d), (n, hkv, d)))
    q[..., 0], k[..., 0] = 4.0, 0.0
    k *= 0.5
    k[0] = 0.0
    k[0, :, 0] = nats * d ** 0.5 / 4.0
    v = 32.0 + 4.0 * v
    v[0] = 0.0
    return (t.to(dtype) for t in (q, k, v))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("nats", [10.0, 16.0, 18.0])
def test_packed_sink(nats, hq, hkv, d, dtype, gpu_device):
    """One key has nearly all of a token's probability and a value of 0: what is left is
    the sum of many small ones."""
    n = 8192
    q, k, v = _sink(n, n, hq, hkv, d, nats, dtype, 3)
    starts = torch.tensor([0, n], dtype=torch.int32, device=gpu_device)
    plan = prepare_packed_gqa(q.to(gpu_device), k.to(gpu_device), v.to(gpu_device), starts)
    _assert_rows(plan.output, q, k, v, lambda r: r + 1, [0, 1, 40, 500, 4095, 4096, 8000, n - 1])
    plan.check_inputs()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("n,width", [(2000, 125), (2000, 20000), (131072, 8192)])
@pytest.mark.parametrize("nats", [10.0, 16.0, 18.0])
def test_paged_sink(nats, n, width, hq, hkv, d, dtype, gpu_device):
    """The same over pages, worked on by teams, by teams in a wide table, and split
    over the keys."""
    rows, page = 3, 16
    q, k, v = _sink(n, rows, hq, hkv, d, nats, dtype, 4)
    pages = [t.view(n // page, page, hkv, d).transpose(1, 2).contiguous().to(gpu_device) for t in (k, v)]
    tables = torch.full((rows, width), -1, dtype=torch.int32)
    tables[:, :n // page] = torch.arange(n // page)
    lengths = [n, n - 37, 40]
    plan = prepare_paged_gqa(q.to(gpu_device), *pages, tables.to(gpu_device),
                             torch.tensor(lengths, dtype=torch.int32, device=gpu_device))
    _assert_rows(plan.output, q, k, v, lambda r: lengths[r], range(rows))
    plan.check_inputs()


def _check_large(q0, scale, negative, dtype, device):
    n, d, page = 640, 64, 16
    g = torch.Generator().manual_seed(5)
    q, k, v = torch.zeros(n, 2, d), torch.zeros(n, 1, d), torch.randn(n, 1, d, generator=g)
    # 16 apart, so that bf16 holds them too; rising slowly, many of them equal.
    q[..., 0] = q0
    k[:, 0, 0] = 2048.0 + 16.0 * (torch.arange(n) // 5 % 60 + torch.randint(0, 3, (n,), generator=g))
    if negative:
        k = -k
    q, k, v = (t.to(dtype) for t in (q, k, v))
    starts = torch.tensor([0, n], dtype=torch.int32, device=device)
    packed = prepare_packed_gqa(q.to(device), k.to(device), v.to(device), starts, scale=scale)
    _assert_rows(packed.output, q, k, v, lambda r: r + 1, range(0, n, 37), scale)
    lengths = list(range(1, n + 1, 37))
    rows = len(lengths)
    pages = [t.view(n // page, page, 1, d).transpose(1, 2).contiguous().to(device) for t in (k, v)]
    for width in (n // page, 20000):
        tables = torch.full((rows, width), -1, dtype=torch.int32)
        tables[:, :n // page] = torch.arange(n // page)
        paged = prepare_paged_gqa(q[:rows].to(device), *pages, tables.to(device),
                                  torch.tensor(lengths, dtype=torch.int32, device=device), scale=scale)
        _assert_rows(paged.output, q, k, v, lambda r: lengths[r], range(rows), scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q0", [1.0, 64.0, 720.0, 2300.0, 4096.0, 16384.0, 61440.0])
@pytest.mark.parametrize("negative", [False, True])
def test_large_scores(negative, q0, dtype, gpu_device):
    """Scores from hundreds to tens of millions, their differences far from 1: the keys
    of the largest one share the probability equally."""
    _check_large(q0, None, negative, dtype, gpu_device)


@pytest.mark.parametrize("dtype,scale", [(torch.bfloat16, 5.75), (torch.float16, 0.36)])
@pytest.mark.parametrize("negative", [False, True])
def test_largest_scores(negative, dtype, scale, gpu_device):
    """The same just below 2^30 (fp16: 2^26), where they are documented to end."""
    assert 0.99 * 2 ** (30 if dtype == torch.bfloat16 else 26) < 61440 * (2048 + 16 * 61) * scale < 2 ** (
        30 if dtype == torch.bfloat16 else 26)
    _check_large(61440.0, scale, negative, dtype, gpu_device)


def test_paged_longest(gpu_device):
    """As many keys as a table may name, 2^31 - 16, all of one page.  Keys of 0 give
    every key the same probability, a power of two, and the waves' sums of values
    of 0 to 3 are whole numbers below 2^24 times that; joining up to 4096 of them
    is off by 2^-12 of the sum at most, less than half a step of bf16, which holds the
    mean itself."""
    page, width = 16, (1 << 27) - 1
    g = torch.Generator().manual_seed(6)
    v = torch.randint(0, 4, (1, 1, page, 64), generator=g).to(torch.bfloat16).to(gpu_device)
    q = torch.ones(1, 1, 64, dtype=torch.bfloat16, device=gpu_device)
    tables = torch.zeros(1, width, dtype=torch.int32, device=gpu_device)
    lengths = torch.tensor([40], dtype=torch.int32, device=gpu_device)
    plan = prepare_paged_gqa(q, torch.zeros_like(v), v, tables, lengths)
    plan.check_inputs()
    mean = v[0, 0].float().mean(0).to(torch.bfloat16)
    for n in (32, page * width - 32, page * width - 16, page * width):
        lengths.fill_(n)
        assert torch.equal(plan.run()[0, 0], mean), n
        plan.check_inputs()
    lengths.fill_(2 ** 31 - 1)      # past the table: taken as all of it
    assert torch.equal(plan.run()[0, 0], mean)
    assert plan.read_status() == N.GQA_STATUS_BAD_BOUNDS
