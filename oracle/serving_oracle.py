"""Plain restatements of the packed and paged attention and of the paged cache,
for the tests: attention in 64 bits, the cache as Python lists taken row by row."""
from __future__ import annotations

import math

import torch


def attention_rows(q, k, v, scale=None):
    """q [Hq, D] over the keys k, v [n, Hkv, D] in 64 bits.  Returns the output
    [Hq, D] and sum p |v| / sum p, which bounds what rounding p can do."""
    hq, d = q.shape
    n, hkv, _ = k.shape
    if n == 0:
        return torch.zeros(hq, d, dtype=torch.float64), torch.zeros(hq, d, dtype=torch.float64)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    kk = k.double().repeat_interleave(hq // hkv, 1).transpose(0, 1)
    vv = v.double().repeat_interleave(hq // hkv, 1).transpose(0, 1)
    p = torch.softmax((kk @ q.double()[:, :, None])[:, :, 0] * scale, dim=1)[:, None, :]
    return (p @ vv)[:, 0], (p @ vv.abs())[:, 0]


def packed_attention(q, k, v, starts, scale=None):
    """Causal attention within each sequence; rows of no sequence are NaN."""
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    group, d = q.shape[1] // k.shape[1], q.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    for a, b in zip(starts[:-1], starts[1:]):
        if a == b:
            continue
        hidden = torch.ones(b - a, b - a, dtype=torch.bool).triu(1)
        for h in range(q.shape[1]):
            kh, vh = k[a:b, h // group].double(), v[a:b, h // group].double()
            s = (q[a:b, h].double() @ kh.t().contiguous()) * scale
            p = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1)
            out[a:b, h], bound[a:b, h] = p @ vh, p @ vh.abs()
    return out, bound


def paged_attention(q, k_pages, v_pages, tables, lengths, scale=None):
    """One token per sequence; k_pages, v_pages [P, Hkv, page, D]."""
    page = k_pages.shape[2]
    outs = []
    for b, n in enumerate(lengths):
        places = [(tables[b][j // page], j % page) for j in range(n)]
        rows = torch.tensor([p for p, _ in places], dtype=torch.long), torch.tensor([r for _, r in places],
                                                                                   dtype=torch.long)
        outs.append(attention_rows(q[b], k_pages[rows[0], :, rows[1]], v_pages[rows[0], :, rows[1]], scale))
    return torch.stack([o for o, _ in outs]), torch.stack([m for _, m in outs])


def tolerance(ref, bound, dtype, keys, vmax):
    """How far a kernel's output may be off.  A rounding to the type is off by at
    most u = eps / 2: once for each probability (u * bound in all) and once for
    the output (u * |ref|, and u^2 for the two together).  Scores of N(0, 1)
    rows of up to 128 elements are off by at most 130 * 2^-24 * sum |q k| * scale
    < 2^-13, probabilities by that and by the exp2 and the sums in fp32: 2^-12 of
    the bound covers them.  fp16 probabilities below 2^-14 are off by 2^-25 each
    against the largest one of at least 2^11, so by 2^-36 of the sum at most."""
    u = torch.finfo(dtype).eps / 2
    small = keys * 2.0 ** -36 * vmax if dtype == torch.float16 else 0.0
    return bound * (u + u * u + 2.0 ** -12) + ref.abs() * u + small


class Cache:
    """The cache's bookkeeping, a row at a time."""

    def __init__(self, pages, page_size, sequences, max_pages, max_tokens):
        self.page, self.max_pages, self.max_tokens = page_size, max_pages, max_tokens
        self.tables = [[] for _ in range(sequences)]
        self.lengths = [0] * sequences
        self.refs = [0] * pages
        self.slots, self.starts = [-1] * max_tokens, [0] * (sequences + 1)
        self.moves = []  # (from, to) of the last call's copied pages
        self.status = 0

    def _pages(self, n):
        return -(-n // self.page)

    def reserve(self, counts, stride=0):
        self.slots, self.starts, self.moves = [-1] * self.max_tokens, [0] * len(self.starts), []
        bad, total = 0, 0
        for n, c in zip(self.lengths, counts):
            if c < 0 or c > self.max_tokens or (stride and c > stride):
                bad |= 16
            elif self._pages(n + c) > self.max_pages:
                bad |= 8
            else:
                total += c
        if total > self.max_tokens:
            bad |= 16
        refs, tables = list(self.refs), [list(t) for t in self.tables]
        moves, starts, slots = [], [0], [-1] * self.max_tokens
        if not bad:
            free = [p for p, r in enumerate(refs) if r == 0]
            for s, (n, c) in enumerate(zip(self.lengths, counts)):
                starts.append(starts[-1] + c)
                if c and n % self.page and refs[tables[s][-1]] > 1:
                    if not free:
                        bad |= 4
                        break
                    old, new = tables[s][-1], free.pop(0)
                    refs[old] -= 1
                    refs[new] = 1
                    tables[s][-1] = new
                    moves.append((old, new))
                while not bad and len(tables[s]) < self._pages(n + c):
                    if not free:
                        bad |= 4
                        break
                    tables[s].append(free.pop(0))
                    refs[tables[s][-1]] = 1
                if bad:
                    break
                for i in range(c):
                    at = s * stride + i if stride else starts[s] + i
                    slots[at] = tables[s][(n + i) // self.page] * self.page + (n + i) % self.page
        self.status |= bad
        if bad:
            return
        self.refs, self.tables, self.moves, self.starts, self.slots = refs, tables, moves, starts, slots
        self.lengths = [n + c for n, c in zip(self.lengths, counts)]

    def fork(self, src, dst):
        rows, lengths, taken = [list(t) for t in self.tables], list(self.lengths), set()
        self.moves = []
        for a, b in zip(src, dst):
            if a < 0 or b < 0:
                continue
            if a >= len(lengths) or b >= len(lengths):
                self.status |= 1
                continue
            if lengths[b] or b in taken:
                self.status |= 2
                continue
            taken.add(b)
            self.tables[b], self.lengths[b] = list(rows[a]), lengths[a]
            for p in rows[a]:
                self.refs[p] += 1

    def free(self, rows):
        self.moves = []
        for r in rows:
            if r >= len(self.lengths):
                self.status |= 1
            elif r >= 0:
                for p in self.tables[r]:
                    self.refs[p] -= 1
                self.tables[r], self.lengths[r] = [], 0

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if not self.refs[p]]
        self.moves = list(zip([p for p in range(used, len(self.refs)) if self.refs[p]], holes))
        to = dict(self.moves)
        for a, b in self.moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.tables = [[to.get(p, p) for p in t] for t in self.tables]

    def check(self):
        """The invariants of the bookkeeping."""
        holders = [0] * len(self.refs)
        for t, n in zip(self.tables, self.lengths):
            assert len(t) == self._pages(n) <= self.max_pages and len(set(t)) == len(t)
            for p in t:
                holders[p] += 1
        assert holders == self.refs


# ---- microscaled rows -----------------------------------------------------------

E4M3 = [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:-1]
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_LAST = {("mxfp8", torch.bfloat16): 119, ("mxfp8", torch.float16): 7, ("mxfp4", torch.bfloat16): 125,
         ("mxfp4", torch.float16): 13}


def mx_quantise(x, storage, dtype):
    """Rows [..., D] of tokens of a type -> element codes uint8 [..., D] and scale
    bytes uint8 [..., D / 32], by search over the table of elements."""
    table = torch.tensor(E4M3 if storage == "mxfp8" else E2M1, dtype=torch.float64)
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, 0.0)
    byte = torch.full(top.shape, 10, dtype=torch.long)
    for e in range(-116, _LAST[storage, dtype] + 1):  # the next larger scale where this one does not do
        byte = torch.where(top > float(table[-1]) * 2.0 ** (e - 1), e + 127, byte)
    y = x / torch.pow(torch.tensor(2.0, dtype=torch.float64), byte - 127)[..., None]
    a = y.abs().clamp(max=float(table[-1]))
    low = torch.searchsorted(table, a, right=True) - 1
    high = (low + 1).clamp(max=len(table) - 1)
    below, above = a - table[low], table[high] - a
    code = torch.where((below > above) | ((below == above) & (low % 2 == 1)), high, low)
    code = torch.where(above == 0, high, code) + torch.signbit(y) * (128 if storage == "mxfp8" else 8)
    byte = torch.where(finite, byte, 255)
    return torch.where(finite[..., None], code, 0).flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def mx_values(codes, scales, storage):
    """What codes [..., D] under scale bytes [..., D / 32] stand for, in 64 bits."""
    table = E4M3 + [math.nan] if storage == "mxfp8" else E2M1
    table = torch.tensor(table + [-a for a in table], dtype=torch.float64)
    power = torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.long() - 127)
    power = torch.where(scales == 255, math.nan, power)
    return (table[codes.long()].unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)


def mx_pack(codes, storage):
    """Codes as they lie in a cache: two of four bits in a byte, the earlier low."""
    return codes if storage == "mxfp8" else codes[..., 0::2] | codes[..., 1::2] << 4


def mx_unpack(held, storage):
    return held if storage == "mxfp8" else torch.stack([held & 15, held >> 4], -1).flatten(-2)


# ---- norm and rotation ------------------------------------------------------------


def norm_rope(x, positions, inv_freq, weight=None, eps=1e-6, interleaved=False):
    """x [N, H, D] in 64 bits, pair by pair; also the magnitude of each pair, which
    bounds what a rotation's roundings can do."""
    x = x.double()
    d, half = x.shape[-1], len(inv_freq)
    if weight is not None:
        x = x * weight.double() / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    out, size = x.clone(), x.abs()
    for i in range(half):
        a = positions.double() * float(inv_freq[i])
        c, s = a.cos()[:, None], a.sin()[:, None]
        low, high = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        out[..., low] = x[..., low] * c - x[..., high] * s
        out[..., high] = x[..., high] * c + x[..., low] * s
        size[..., low] = size[..., high] = x[..., low].abs() + x[..., high].abs()
    return out, size
