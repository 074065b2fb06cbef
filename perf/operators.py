"""Operators of a paged key-value cache and the attention around it, measured.

Four kinds of case, each one step of a serving program:

* ``prompt``: causal attention of several prompts packed behind each other
  (``prepare_packed_gqa``);
* ``decode``: attention of one new token per sequence over the pages of a cache
  (``prepare_paged_gqa``);
* ``append``: keys and values of new tokens written to their slots
  (``PagedKVCache.append``);
* ``fork`` and ``compact``: sequences forked, extended by one token with
  copy-on-write and freed again (``fork``, ``reserve``, ``free``), and the pages
  in use moved to the front (``compact``).

``own`` selects the framework's kernels; otherwise ``run`` computes the same
with elementary torch operations in 32 bits.  Lengths depend on the case alone,
page numbers and values on the seed.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _prompt(name, seqs, low, high, heads=32, kv_heads=8, dim=128, dtype="bf16", fused=False):
    case = dict(kind="prompt", S=seqs, low=low, high=high, Hq=heads, Hkv=kv_heads, D=dim, dtype=dtype, fused=fused)
    return dict(case, name=name) if name else case


def _decode(name, seqs, low, high, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16):
    case = dict(kind="decode", S=seqs, low=low, high=high, Hq=heads, Hkv=kv_heads, D=dim, dtype=dtype, page=page)
    return dict(case, name=name) if name else case


def _append(name, tokens, pages, kv_heads=8, dim=128, dtype="bf16", page=16, fused=False):
    case = dict(kind="append", N=tokens, pages=pages, Hkv=kv_heads, D=dim, dtype=dtype, page=page, fused=fused)
    return dict(case, name=name) if name else case


def _fork(name, parents, children, low, high, layers=2, kv_heads=8, dim=128, dtype="bf16", page=16):
    case = dict(kind="fork", S=parents, children=children, low=low, high=high, layers=layers, Hkv=kv_heads, D=dim,
                dtype=dtype, page=page)
    return dict(case, name=name) if name else case


def _compact(name, seqs, low, high, layers=2, kv_heads=8, dim=128, dtype="bf16", page=16):
    case = dict(kind="compact", S=seqs, low=low, high=high, layers=layers, Hkv=kv_heads, D=dim, dtype=dtype, page=page)
    return dict(case, name=name) if name else case


def listed():
    return [
        # A few short chat turns: latency.
        _prompt("prompt-small", 4, 1, 48),
        # A batch of ordinary ragged prompts, q, k and v views of one projection.
        _prompt("prompt-ragged", 16, 64, 2048, fused=True),
        # One long document.
        _prompt("prompt-long", 1, 16384, 16384),
        # A smaller model in half precision: heads of 64, three per key head.
        _prompt("prompt-fp16-d64", 8, 300, 1500, heads=12, kv_heads=4, dim=64, dtype="fp16"),
        # One short conversation: latency.
        _decode("decode-one", 1, 700, 700),
        # A batch of conversations of every age.
        _decode("decode-ragged", 64, 1, 8192),
        # One very long context, split over its length.
        _decode("decode-long", 1, 131072, 131072),
        # Many short contexts of a smaller model in half precision, large pages.
        _decode("decode-fp16-d64", 200, 16, 2000, heads=14, kv_heads=2, dim=64, dtype="fp16", page=64),
        # The write of a decode step and of a prefill chunk.
        _append("append-step", 64, 1024),
        _append("append-chunk", 8191, 1024, fused=True),
        # Parallel sampling: three more samples of each prompt start.
        _fork("fork-step", 32, 3, 100, 4000),
        # A fragmented cache after many sequences have left.
        _compact("compact", 48, 100, 2000, layers=4),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "decode", "decode", "append", "fork", "compact"])
    heads, kv, dim = rng.choice([(32, 8, 128), (16, 8, 128), (4, 4, 128), (8, 1, 128), (12, 4, 64), (14, 2, 64), (6, 6, 64)])
    dtype, page = rng.choice(["bf16", "fp16"]), rng.choice([16, 32, 64, 80])
    if kind == "prompt":
        seqs = _log_int(rng, 1, 32)
        high = _log_int(rng, 1, 8192 // math.isqrt(seqs))
        return _prompt(None, seqs, _log_int(rng, 1, high), high, heads, kv, dim, dtype, rng.random() < 0.5)
    if kind == "decode":
        seqs = _log_int(rng, 1, 256)
        high = _log_int(rng, 1, min(65536, 200000 // seqs))
        return _decode(None, seqs, _log_int(rng, 1, high), high, heads, kv, dim, dtype, page)
    if kind == "append":
        tokens = _log_int(rng, 1, 8191)
        return _append(None, tokens, _log_int(rng, -(-tokens // page), 1024), kv, dim, dtype, page, rng.random() < 0.5)
    seqs = _log_int(rng, 1, 48)
    high = _log_int(rng, 1, 2000)
    low, layers = _log_int(rng, 1, high), rng.randint(1, 3)
    if kind == "fork":
        return _fork(None, min(seqs, 32), rng.randint(1, 3), low, high, layers, kv, dim, dtype, page)
    return _compact(None, seqs, low, high, layers, kv, dim, dtype, page)


# ---- inputs -----------------------------------------------------------------


def _lengths(case):
    """Sequence lengths, spread over the logarithm of the case's range."""
    rng = random.Random(f"{case['S']} {case['low']} {case['high']}")
    return [_log_int(rng, case["low"], case["high"]) for _ in range(case["S"])]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _fill(t, gen, scale=1.0):
    """N(0, scale) into a tensor, in pieces along the first dimension."""
    rows = max(1, (1 << 26) // max(1, math.prod(t.shape[1:])))
    for i in range(0, t.shape[0], rows):
        part = t[i:i + rows]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * scale)
    return t


def _rows(case, tokens, gen, query=True):
    """q, k and v of some tokens: three tensors, or views of one projection."""
    dtype, d, kv = DTYPES[case["dtype"]], case["D"], case["Hkv"]
    counts = [case["Hq"], kv, kv] if query else [kv, kv]
    if case["fused"]:
        row = _fill(torch.empty((tokens, sum(counts), d), dtype=dtype, device="cuda"), gen)
        parts = row.split(counts, dim=1)
    else:
        parts = [_fill(torch.empty((tokens, c, d), dtype=dtype, device="cuda"), gen) for c in counts]
    return parts


def _starts(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths) + 1)]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(lengths, page, pages, width, seed):
    """Rows of page numbers drawn without order, -1 behind the last page."""
    order = list(range(pages))
    random.Random(int(seed) * 7919 + pages).shuffle(order)
    rows, at = [], 0
    for length in lengths:
        n = -(-length // page)
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return rows


def _cache(case, pages, width, sequences, tokens, layers):
    """The cache of a program: the framework's, or the same tensors by themselves."""
    kv, page, d, dtype = case["Hkv"], case["page"], case["D"], DTYPES[case["dtype"]]
    if own:
        from llm_gpu_kernels_amd import PagedKVCache
        return PagedKVCache(pages, page, kv, d, sequences=sequences, max_pages=width, max_tokens=tokens, layers=layers,
                            dtype=dtype, device="cuda")

    class Tensors:
        pass

    c = Tensors()
    c.k, c.v = (torch.empty((layers, pages, kv, page, d), dtype=dtype, device="cuda") for _ in range(2))
    c.tables = torch.full((sequences, width), -1, dtype=torch.int32, device="cuda")
    c.lengths = torch.zeros(sequences, dtype=torch.int32, device="cuda")
    c.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    c.slots = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
    c.starts = torch.zeros(sequences + 1, dtype=torch.int32, device="cuda")
    return c


def _fill_cache(cache, gen):
    for layer in range(cache.k.shape[0]):
        _fill(cache.k[layer], gen)
        _fill(cache.v[layer], gen)


def _prompt_inputs(case, seed):
    lengths = _lengths(case)
    q, k, v = _rows(case, sum(lengths), _generator(seed))
    return lengths, q, k, v


def _decode_inputs(case, seed):
    gen = _generator(seed)
    lengths, page, dtype = _lengths(case), case["page"], DTYPES[case["dtype"]]
    width = -(-max(lengths) // page) + 1
    pages = sum(-(-n // page) for n in lengths) + 3
    k, v = (_fill(torch.empty((pages, case["Hkv"], page, case["D"]), dtype=dtype, device="cuda"), gen) for _ in range(2))
    q = _fill(torch.empty((case["S"], case["Hq"], case["D"]), dtype=dtype, device="cuda"), gen, 1.5)
    return lengths, q, k, v, _tables(lengths, page, pages, width, seed)


def _append_inputs(case, seed):
    k, v = _rows(case, case["N"], _generator(seed), query=False)
    slots = random.Random(int(seed) + 1).sample(range(case["pages"] * case["page"]), case["N"])
    return k, v, slots


def _fork_inputs(case, seed):
    """Parents in the first rows, the others empty; page numbers without order."""
    lengths, page, n = _lengths(case), case["page"], case["children"]
    sequences = case["S"] * (n + 1)
    width = -(-max(lengths) // page) + 1
    used = sum(-(-x // page) for x in lengths)
    pages = used + 2 * sequences
    tables = _tables(lengths, page, pages, width, seed) + [[-1] * width] * (sequences - case["S"])
    src = [i for i in range(case["S"]) for _ in range(n)]
    dst = list(range(case["S"], sequences))
    return dict(lengths=lengths + [0] * len(dst), tables=tables, pages=pages, width=width, sequences=sequences, src=src,
                dst=dst, counts=[0] * case["S"] + [1] * len(dst))


def _compact_inputs(case, seed):
    lengths, page = _lengths(case), case["page"]
    pages = 2 * sum(-(-x // page) for x in lengths) + 5
    width = -(-max(lengths) // page)
    return dict(lengths=lengths, tables=_tables(lengths, page, pages, width, seed), pages=pages, width=width,
                sequences=case["S"])


def _refs(tables, pages):
    refs = [0] * pages
    for row in tables:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return refs


def prepare(case, seed):
    kind, gen = case["kind"], _generator(int(seed) + 12345)
    state = dict(case=case)
    if kind == "prompt":
        lengths, q, k, v = _prompt_inputs(case, seed)
        starts = _int32(_starts(lengths))
        if own:
            from llm_gpu_kernels_amd import prepare_packed_gqa
            return dict(state, plan=prepare_packed_gqa(q, k, v, starts))
        return dict(state, q=q, k=k, v=v, lengths=lengths)
    if kind == "decode":
        lengths, q, k, v, tables = _decode_inputs(case, seed)
        tables, on_gpu = _int32(tables), _int32(lengths)
        if own:
            from llm_gpu_kernels_amd import prepare_paged_gqa
            return dict(state, plan=prepare_paged_gqa(q, k, v, tables, on_gpu))
        return dict(state, q=q, k=k, v=v, tables=tables, lengths=lengths)
    if kind == "append":
        k, v, slots = _append_inputs(case, seed)
        cache = _cache(case, case["pages"], case["pages"], 1, case["N"], 1)
        cache.slots.copy_(torch.tensor(slots, device="cuda"))
        _fill_cache(cache, gen)
        return dict(state, cache=cache, k=k, v=v)
    x = _fork_inputs(case, seed) if kind == "fork" else _compact_inputs(case, seed)
    cache = _cache(case, x["pages"], x["width"], x["sequences"], x["sequences"], case["layers"])
    _fill_cache(cache, gen)
    cache.tables.copy_(_int32(x["tables"]))
    cache.lengths.copy_(_int32(x["lengths"]))
    cache.refs.copy_(_int32(_refs(x["tables"], x["pages"])))
    if kind == "fork":
        return dict(state, cache=cache, src=_int32(x["src"]), dst=_int32(x["dst"]), counts=_int32(x["counts"]))
    return dict(state, cache=cache, tables=cache.tables.clone(), refs=cache.refs.clone())


# ---- one pass -----------------------------------------------------------------


def _attend(q, k, v, lengths_of_rows=None):
    """Softmax attention of one key head's queries [n, group, D] over its keys
    [m, D]; a row sees its first ``lengths_of_rows`` keys, or all."""
    n, group, d = q.shape
    s = (q.reshape(-1, d) @ k.t().contiguous()).view(n, group, -1) / math.sqrt(d)
    if lengths_of_rows is not None:
        hidden = torch.arange(k.shape[0], device="cuda") >= lengths_of_rows[:, None]
        s.masked_fill_(hidden[:, None, :], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    s /= s.sum(-1, keepdim=True)
    return (s.view(n * group, -1) @ v).view(n, group, d)


def _prompt_attention(lengths, q, k, v, wide):
    """Causal attention of every sequence by itself, in the type ``wide``."""
    out = torch.empty(q.shape, dtype=wide, device="cuda")
    kv, at = k.shape[1], 0
    group = q.shape[1] // kv
    for n in lengths:
        rows = max(1, (1 << 27) // (group * n))
        for j in range(kv):
            kj, vj = k[at:at + n, j].to(wide), v[at:at + n, j].to(wide)
            for i in range(0, n, rows):
                m = min(n, i + rows)
                seen = torch.arange(i + 1, m + 1, device="cuda")
                out[at + i:at + m, j * group:(j + 1) * group] = _attend(
                    q[at + i:at + m, j * group:(j + 1) * group].to(wide), kj[:m], vj[:m], seen)
        at += n
    return out


def _decode_attention(lengths, q, k, v, tables, wide):
    out = torch.zeros(q.shape, dtype=wide, device="cuda")
    kv, page, d = k.shape[1:]
    group = q.shape[1] // kv
    for b, n in enumerate(lengths):
        rows = tables[b, :-(-n // page)].long()
        for j in range(kv):
            kj, vj = (t[rows, j].reshape(-1, d)[:n].to(wide) for t in (k, v))
            out[b, j * group:(j + 1) * group] = _attend(q[b:b + 1, j * group:(j + 1) * group].to(wide), kj, vj)[0]
    return out


def _plain_free(c, rows, page):
    rows = rows.long().unique()
    pages = c.tables[rows]
    c.refs.index_add_(0, pages[pages >= 0].long(), -torch.ones_like(pages[pages >= 0]))
    c.tables[rows] = -1
    c.lengths[rows] = 0


def _plain_fork(c, src, dst, page):
    src, dst = src.long(), dst.long()
    pages = c.tables[src]
    c.tables[dst] = pages
    c.lengths[dst] = c.lengths[src]
    c.refs.index_add_(0, pages[pages >= 0].long(), torch.ones_like(pages[pages >= 0]))


def _plain_reserve(c, counts, stride, page):
    length, counts = c.lengths.long(), counts.long()
    row = torch.arange(len(length), device="cuda")
    used, new = (length + page - 1) // page, length + counts
    last = c.tables[row, (length // page).clamp(max=c.tables.shape[1] - 1)].long()
    last = torch.where((counts > 0) & (length % page > 0), last, 0)
    shared = (counts > 0) & (length % page > 0) & (c.refs[last] > 1)
    holders = torch.zeros_like(c.refs).index_add_(0, last[shared], torch.ones_like(c.refs[last[shared]]))
    highest = torch.full_like(c.refs, -1).long().scatter_reduce_(0, last[shared], row[shared], "amax")
    copied = shared & ~((holders[last] == c.refs[last]) & (highest[last] == row))
    need = (new + page - 1) // page - used + copied
    first = need.cumsum(0) - need
    free = (c.refs == 0).nonzero()[:, 0]
    owner = torch.repeat_interleave(row, need)
    free, j = free[:len(owner)], torch.arange(len(owner), device="cuda") - first[owner]
    column = used[owner] + j - copied[owner].long()
    c.tables[owner, column] = free.to(torch.int32)
    c.refs[free] = 1
    c.refs.index_add_(0, last[copied], -torch.ones_like(c.refs[last[copied]]))
    target = c.tables[row[copied], (length // page)[copied]].long()
    c.k[:, target] = c.k[:, last[copied]]
    c.v[:, target] = c.v[:, last[copied]]
    c.lengths.copy_(new)
    c.starts[1:] = counts.cumsum(0)
    c.slots.fill_(-1)
    token = torch.repeat_interleave(row, counts)
    i = torch.arange(len(token), device="cuda") - c.starts[token].long()
    position = length[token] + i
    place = token * stride + i if stride else c.starts[token].long() + i
    c.slots[place] = c.tables[token, position // page].long() * page + position % page


def _plain_compact(c):
    used = c.refs > 0
    n = used.sum()
    below = torch.arange(len(used), device="cuda") < n
    to, source = (below & ~used).nonzero()[:, 0], (~below & used).nonzero()[:, 0]
    moved = torch.arange(len(used), device="cuda")
    moved[source] = to
    c.k[:, to] = c.k[:, source]
    c.v[:, to] = c.v[:, source]
    c.refs[to] = c.refs[source]
    c.refs[source] = 0
    c.tables.copy_(torch.where(c.tables >= 0, moved[c.tables.long().clamp(min=0)].to(torch.int32), c.tables))


def run(state):
    case = state["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind in ("prompt", "decode"):
        if own:
            return state["plan"].run()
        if kind == "prompt":
            return _prompt_attention(state["lengths"], state["q"], state["k"], state["v"], torch.float32).to(dtype)
        return _decode_attention(state["lengths"], state["q"], state["k"], state["v"], state["tables"],
                                 torch.float32).to(dtype)
    c = state["cache"]
    if kind == "append":
        if own:
            c.append(0, state["k"], state["v"])
        else:
            page, offset = c.slots // case["page"], c.slots % case["page"]
            c.k[0][page, :, offset] = state["k"]
            c.v[0][page, :, offset] = state["v"]
        return dict(k=c.k, v=c.v)
    if kind == "fork":
        # The samples of the pass before leave, new ones start and take a token.
        if own:
            c.free(state["dst"])
            c.fork(state["src"], state["dst"])
            c.reserve(state["counts"], stride=1)
        else:
            _plain_free(c, state["dst"], case["page"])
            _plain_fork(c, state["src"], state["dst"], case["page"])
            _plain_reserve(c, state["counts"], 1, case["page"])
        return dict(tables=c.tables, lengths=c.lengths, refs=c.refs, slots=c.slots, starts=c.starts, k=c.k, v=c.v)
    # The cache is fragmented again first (a program's comes so from its use).
    c.tables.copy_(state["tables"])
    c.refs.copy_(state["refs"])
    if own:
        c.compact()
    else:
        _plain_compact(c)
    return dict(tables=c.tables, lengths=c.lengths, refs=c.refs, k=c.k, v=c.v)


# ---- what a pass cannot do without ----------------------------------------------


def work(case):
    kind, kv, d = case["kind"], case["Hkv"], case["D"]
    row = kv * d * 2  # bytes of one token's keys or values
    if kind == "append":
        return dict(bytes=case["N"] * (4 * row + 8), flops=0)
    lengths = _lengths(case)
    if kind == "prompt":
        return dict(bytes=sum(lengths) * 2 * (row + case["Hq"] * d * 2) + 4 * (len(lengths) + 1),
                    flops=2 * case["Hq"] * d * sum(n * (n + 1) for n in lengths))
    pages = sum(-(-n // case["page"]) for n in lengths)
    if kind == "decode":
        return dict(bytes=sum(lengths) * 2 * row + case["S"] * (case["Hq"] * d * 4 + 4) + 4 * pages,
                    flops=4 * case["Hq"] * d * sum(lengths))
    one = 2 * case["layers"] * row * case["page"]  # bytes of a page in every layer, keys and values
    if kind == "fork":
        # Tables: read and written by the fork, read by the free that undoes it.
        copies = sum(n % case["page"] > 0 for n in lengths) * case["children"]
        return dict(bytes=2 * one * copies + 5 * 4 * pages * case["children"], flops=0)
    # Half of the pages in use lie behind the place where they end up.
    total = 2 * pages + 5
    moved = pages * (total - pages) // total
    return dict(bytes=2 * one * moved + 8 * total + 8 * pages, flops=0)


# ---- the same in 64 bits ----------------------------------------------------------


def _exact_rows(q, k, v, seen):
    """One key head in 64 bits: queries [n, group, D], the row i sees the first
    seen[i] keys."""
    n, group, d = q.shape
    scores = torch.matmul(q.reshape(n * group, d), k.transpose(0, 1).contiguous()).mul_(d ** -0.5)
    index = torch.arange(k.shape[0], device="cuda").expand(n * group, -1)
    scores = torch.where(index < seen.repeat_interleave(group)[:, None], scores, -math.inf)
    return torch.matmul(torch.softmax(scores, dim=1), v).view(n, group, d)


def _exact_attention(case, seed):
    if case["kind"] == "prompt":
        lengths, q, k, v = _prompt_inputs(case, seed)
    else:
        lengths, q, pk, pv, tables = _decode_inputs(case, seed)
    group = case["Hq"] // case["Hkv"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, n in enumerate(lengths):
        if case["kind"] == "decode":
            places = torch.tensor([tables[b][t // case["page"]] * case["page"] + t % case["page"] for t in range(n)],
                                  device="cuda")
        for h in range(case["Hkv"]):
            heads = slice(h * group, (h + 1) * group)
            if case["kind"] == "decode":
                kh, vh = (t[places // case["page"], h, places % case["page"]].double() for t in (pk, pv))
                out[b, heads] = _exact_rows(q[b:b + 1, heads].double(), kh, vh, torch.tensor([n], device="cuda"))[0]
                continue
            kh, vh = k[first:first + n, h].double(), v[first:first + n, h].double()
            step = max(1, (1 << 26) // (group * n))
            for i in range(0, n, step):
                rows = range(i, min(n, i + step))
                out[first + i:first + rows.stop, heads] = _exact_rows(
                    q[first + i:first + rows.stop, heads].double(), kh, vh,
                    torch.tensor([r + 1 for r in rows], device="cuda"))
        first += n
    return out


def _exact_values(case, seed, pages, tokens, layers):
    """The cache's keys and values as prepared, [layers, pages, ...]."""
    dtype = DTYPES[case["dtype"]]
    k, v = (torch.empty((layers, pages, case["Hkv"], case["page"], case["D"]), dtype=dtype, device="cuda")
            for _ in range(2))
    gen = _generator(int(seed) + 12345)
    for layer in range(layers):
        _fill(k[layer], gen)
        _fill(v[layer], gen)
    return k, v


def _moved(t, moves):
    """Pages ``to`` hold what ``source`` held, for every (source, to)."""
    if moves:
        source, to = (torch.tensor(x, device="cuda") for x in zip(*moves))
        t = t.index_copy(1, to, t.index_select(1, source))
    return t


def exact(case, seed):
    kind = case["kind"]
    if kind in ("prompt", "decode"):
        return _exact_attention(case, seed)
    if kind == "append":
        k, v, slots = _append_inputs(case, seed)
        out = []
        for cache, rows in zip(_exact_values(case, seed, case["pages"], case["N"], 1), (k, v)):
            flat = cache[0].transpose(1, 2).reshape(-1, case["Hkv"], case["D"])
            flat = flat.index_copy(0, torch.tensor(slots, device="cuda"), rows.contiguous())
            out.append(flat.view(case["pages"], case["page"], case["Hkv"], case["D"]).transpose(1, 2)[None].double())
        return dict(k=out[0], v=out[1])
    page = case["page"]
    x = _fork_inputs(case, seed) if kind == "fork" else _compact_inputs(case, seed)
    tables, lengths = [list(row) for row in x["tables"]], list(x["lengths"])
    refs, moves = _refs(tables, x["pages"]), []
    k, v = _exact_values(case, seed, x["pages"], x["sequences"], case["layers"])
    if kind == "compact":
        used = sum(r > 0 for r in refs)
        holes = [p for p in range(used) if not refs[p]]
        moves = list(zip([p for p in range(used, len(refs)) if refs[p]], holes))
        where = dict(moves)
        tables = [[where.get(p, p) for p in row] for row in tables]
        k, v = _moved(k, moves).double(), _moved(v, moves).double()
        return dict(tables=_int32(tables), lengths=_int32(lengths), refs=_int32(_refs(tables, len(refs))), k=k, v=v)
    for a, b in zip(x["src"], x["dst"]):
        tables[b], lengths[b] = list(tables[a]), lengths[a]
        for p in tables[b]:
            if p >= 0:
                refs[p] += 1
    slots, starts = [], [0]
    for s, count in enumerate(x["counts"]):
        starts.append(starts[-1] + count)
        if not count:
            slots.append(-1)
            continue
        at = lengths[s] // page
        if lengths[s] % page == 0:
            tables[s][at] = refs.index(0)
            refs[tables[s][at]] = 1
        elif refs[tables[s][at]] > 1:
            to = refs.index(0)
            moves.append((tables[s][at], to))
            refs[tables[s][at]] -= 1
            refs[to] = 1
            tables[s][at] = to
        slots.append(tables[s][at] * page + lengths[s] % page)
        lengths[s] += 1
    return dict(tables=_int32(tables), lengths=_int32(lengths), refs=_int32(refs),
                slots=torch.tensor(slots, device="cuda"), starts=_int32(starts),
                k=_moved(k, moves).double(), v=_moved(v, moves).double())
