"""Operators around a paged key-value cache that is held in few bits or shared.

Kinds of case, each one call of a serving program:

* ``rope``: norms of queries and keys for each head and the rotation by position
  in one pass, with the keys and values written to a cache or not
  (``prepare_qk_norm_rope``);
* ``append``, ``store`` and ``read``: keys and values of new tokens quantised as
  they are written to their slots (``PagedKVCache(storage=...).append``), the
  same and read back, and whole rows read back (``PagedKVCache.gather``);
* ``decode``: attention of one new token per sequence over the pages of such a
  cache (``prepare_paged_gqa`` with scales);
* ``shared``: attention of one new token per sequence where groups of sequences
  start with the same keys (``prepare_shared_gqa``).

Storage ``mxfp8`` holds e4m3 elements and ``mxfp4`` e2m1 elements, two in a byte,
the earlier in the low half; 32 neighbouring elements of a row have one scale, a
power of two in e8m0: the smallest with which all of them are in range.

``own`` selects the framework's kernels; otherwise ``run`` computes the same with
elementary torch operations in 32 bits (angles in 64).  Lengths depend on the
case alone, page numbers, positions and values on the seed.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 32                                    # elements with one scale
LARGEST = {"mxfp8": (1.75, 8), "mxfp4": (1.5, 2)}  # largest element: mantissa, exponent
# Scales go up to where the largest element times the scale is the largest such
# product that is finite in the tokens' type.
LAST_EXPONENT = {("mxfp8", "bf16"): 119, ("mxfp8", "fp16"): 7, ("mxfp4", "bf16"): 125, ("mxfp4", "fp16"): 13}
FIRST_EXPONENT = -117
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _named(case, name):
    return dict(case, name=name) if name else case


def _rope(name, tokens, store="rows", heads=32, kv_heads=8, dim=128, rotary=128, dtype="bf16", norm=True, neighbours=False,
          fused=True, page=16):
    return _named(dict(kind="rope", N=tokens, store=store, Hq=heads, Hkv=kv_heads, D=dim, R=rotary, dtype=dtype, norm=norm,
                       neighbours=neighbours, fused=fused, page=page), name)


def _write(kind, name, tokens, storage, kv_heads=8, dim=128, dtype="bf16", page=16, fused=False):
    return _named(dict(kind=kind, N=tokens, storage=storage, Hkv=kv_heads, D=dim, dtype=dtype, page=page, fused=fused), name)


def _read(name, seqs, low, high, storage, kv_heads=8, dim=128, dtype="bf16", page=16):
    return _named(dict(kind="read", S=seqs, low=low, high=high, storage=storage, Hkv=kv_heads, D=dim, dtype=dtype, page=page),
                  name)


def _decode(name, seqs, low, high, storage, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16):
    return _named(dict(kind="decode", S=seqs, low=low, high=high, storage=storage, Hq=heads, Hkv=kv_heads, D=dim, dtype=dtype,
                       page=page), name)


def _shared(name, groups, few, many, low, high, tail, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16):
    """Groups of few to many sequences, prefixes of low to high keys, 1 to tail keys of a sequence's own."""
    return _named(dict(kind="shared", G=groups, few=few, many=many, low=low, high=high, tail=tail, Hq=heads, Hkv=kv_heads,
                       D=dim, dtype=dtype, page=page), name)


def listed():
    return [
        # The queries and keys of a decode step: latency.
        _rope("rope-step", 16),
        # Those of a long prefill chunk, views of one projection, read by prompt attention.
        _rope("rope-chunk", 8191),
        # A chunk of a smaller model in half precision whose keys go straight into a
        # quantised cache, neighbouring elements rotated, half of each head.
        _rope("rope-into-mxfp8", 2500, store="mxfp8", heads=12, kv_heads=4, dim=64, rotary=32, dtype="fp16", neighbours=True),
        # The write of a decode step and of a prefill chunk, eight bits.
        _write("append", "append-mxfp8-step", 64, "mxfp8"),
        _write("append", "append-mxfp8-chunk", 8191, "mxfp8", fused=True),
        # A chunk written in four bits and read back for the attention of the next one.
        _write("store", "store-mxfp4", 4000, "mxfp4"),
        # The histories of a few conversations read back before prompts that continue them.
        _read("read-mxfp8", 6, 1000, 9000, "mxfp8"),
        # One short conversation: latency.
        _decode("decode-mxfp8-one", 1, 700, 700, "mxfp8"),
        # A batch of conversations of every age.
        _decode("decode-mxfp8-ragged", 64, 1, 8192, "mxfp8"),
        # One very long context in four bits, split over its length.
        _decode("decode-mxfp4-long", 1, 131072, 131072, "mxfp4"),
        # Samples of one question behind an ordinary prompt.
        _shared("shared-samples", 1, 8, 8, 1500, 1500, 100),
        # Several long instructions, each shared by a batch of users.
        _shared("shared-batch", 4, 20, 44, 4000, 12000, 600),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "append", "store", "read", "decode", "decode", "shared", "shared"])
    heads, kv, dim = rng.choice([(32, 8, 128), (16, 8, 128), (4, 4, 128), (8, 1, 128), (12, 4, 64), (14, 2, 64), (6, 6, 64)])
    dtype, page, storage = rng.choice(["bf16", "fp16"]), rng.choice([16, 32, 64, 80]), rng.choice(["mxfp8", "mxfp4"])
    if kind == "rope":
        rotary = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        return _rope(None, _log_int(rng, 1, 8191), rng.choice(["rows", "rows", "pages", "mxfp8"]), heads, kv, dim, rotary,
                     dtype, rng.random() < 0.7, rng.random() < 0.4, rng.random() < 0.7, page)
    if kind in ("append", "store"):
        # Elements of four bits have no values of their own in torch: they are read back.
        return _write(kind, None, _log_int(rng, 1, 8191), "mxfp8" if kind == "append" else storage, kv, dim, dtype, page,
                      rng.random() < 0.5)
    if kind == "read":
        high = _log_int(rng, 1, 9000)
        return _read(None, _log_int(rng, 1, 6), _log_int(rng, 1, high), high, storage, kv, dim, dtype, page)
    if kind == "decode":
        seqs = _log_int(rng, 1, 256)
        high = _log_int(rng, 1, min(65536, 200000 // seqs))
        return _decode(None, seqs, _log_int(rng, 1, high), high, storage, heads, kv, dim, dtype, page)
    groups = _log_int(rng, 1, 4)
    many, high = _log_int(rng, 1, 44), _log_int(rng, 1, 12000)
    return _shared(None, groups, _log_int(rng, 1, many), many, _log_int(rng, 1, high), high, _log_int(rng, 1, 600), heads, kv,
                   dim, dtype, page)


# ---- inputs -----------------------------------------------------------------


def _spread(case, count, low, high, what):
    """Numbers spread over the logarithm of a range, by the case alone."""
    rng = random.Random(f"{what} {count} {low} {high}")
    return [_log_int(rng, low, high) for _ in range(count)]


def _lengths(case):
    return _spread(case, case["S"], case["low"], case["high"], "lengths")


def _groups(case):
    """Members and prefix of every group, the length of every sequence."""
    members = _spread(case, case["G"], case["few"], case["many"], "members")
    prefixes = _spread(case, case["G"], case["low"], case["high"], "prefixes")
    tails = _spread(case, sum(members), 1, case["tail"], "tails")
    owner = [g for g, n in enumerate(members) for _ in range(n)]
    return members, prefixes, [prefixes[g] + t for g, t in zip(owner, tails)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(shape, gen, dtype, scale=1.0):
    """N(0, scale), in pieces along the first dimension."""
    t = torch.empty(shape, dtype=dtype, device="cuda")
    rows = max(1, (1 << 26) // max(1, math.prod(shape[1:])))
    for i in range(0, shape[0], rows):
        part = t[i:i + rows]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * scale)
    return t


def _rows(case, gen, counts):
    """Rows of heads for some tokens: separate tensors, or views of one projection."""
    d, n, dtype = case["D"], case["N"], DTYPES[case["dtype"]]
    if case["fused"]:
        return list(_randn((n, sum(counts), d), gen, dtype).split(counts, dim=1))
    return [_randn((n, c, d), gen, dtype) for c in counts]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


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


def _slots(case, seed):
    """A slot for every token, and the pages they are in: a chunk's tokens fill pages
    one after the other, those of a step belong to as many sequences."""
    page, n, rng = case["page"], case["N"], random.Random(int(seed) + 1)
    pages = -(-n // page) + 2
    order = rng.sample(range(pages), pages)
    if n <= 256 and case["kind"] != "store":
        return rng.sample(range(pages * page), n), pages, order
    return [order[i // page] * page + i % page for i in range(n)], pages, order


def _values(case, seed, pages):
    """Keys and values of all pages before they are quantised."""
    gen = _generator(seed)
    shape = (pages, case["Hkv"], case["page"], case["D"])
    return [_randn(shape, gen, DTYPES[case["dtype"]]) for _ in range(2)]


def _rope_inputs(case, seed):
    gen = _generator(seed)
    d, n, dtype = case["D"], case["N"], DTYPES[case["dtype"]]
    q, k, v = _rows(case, gen, [case["Hq"], case["Hkv"], case["Hkv"]])
    # A chunk continues one far sequence, a step has one token of each of many.
    rng = random.Random(int(seed) + 3)
    first = rng.randrange(120000)
    positions = _int32([first + i for i in range(n)] if n > 256 else [rng.randrange(131072) for _ in range(n)])
    half = case["R"] // 2
    inv_freq = torch.tensor([1e6 ** (-i / half) for i in range(half)], dtype=torch.float32, device="cuda")
    weights = [(1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype) if case["norm"] else None for _ in range(2)]
    return q, k, v, positions, inv_freq, weights


def _paged_inputs(case, seed):
    lengths, page = _lengths(case), case["page"]
    pages = sum(-(-n // page) for n in lengths) + 3
    width = -(-max(lengths) // page) + 1
    return lengths, pages, width, _tables(lengths, page, pages, width, seed)


def _shared_inputs(case, seed):
    members, prefixes, lengths = _groups(case)
    page = case["page"]
    gen = _generator(seed)
    # Whole pages of a prefix are held once; a sequence's own begin with the page where the prefix ends.
    own_pages, at = [], 0
    for n, prefix in zip(members, prefixes):
        whole = prefix // page
        own_pages.append(whole)
        own_pages += [-(-length // page) - whole for length in lengths[at:at + n]]
        at += n
    pages, width = sum(own_pages) + 3, -(-max(lengths) // page) + 1
    parts = iter(_tables([x * page for x in own_pages], page, pages, width, seed))
    k, v = _values(case, int(seed) + 5, pages)
    tables = []
    for n, prefix in zip(members, prefixes):
        first = next(parts)[:prefix // page]
        for i in range(n):
            row = (first + next(parts))[:width]
            tables.append(row)
            rest, head = prefix % page, tables[-1 - i]
            if i and rest:  # the copy that a sequence has of a page that it shared in part
                for t in (k, v):
                    t[row[prefix // page], :, :rest] = t[head[prefix // page], :, :rest]
    q = _randn((len(lengths), case["Hq"], case["D"]), gen, DTYPES[case["dtype"]], 1.5)
    return q, k, v, tables, lengths, members, prefixes


def _cache(case, pages, width, sequences, tokens, storage):
    """The cache of a program: the framework's, or the same tensors by themselves."""
    kv, page, d, dtype = case["Hkv"], case["page"], case["D"], DTYPES[case["dtype"]]
    if own:
        from llm_gpu_kernels_amd import PagedKVCache
        return PagedKVCache(pages, page, kv, d, sequences=sequences, max_pages=width, max_tokens=tokens, dtype=dtype,
                            storage=storage, device="cuda")

    class Tensors:
        pass

    c = Tensors()
    if storage is None:
        c.k, c.v = (torch.zeros((1, pages, kv, page, d), dtype=dtype, device="cuda") for _ in range(2))
    else:
        c.k, c.v = (_elements(torch.zeros((1, pages, kv, page, d if storage == "mxfp8" else d // 2), dtype=torch.uint8,
                                          device="cuda"), storage) for _ in range(2))
        c.k_scales, c.v_scales = (torch.zeros((1, pages, kv, d // BLOCK, page), dtype=torch.uint8, device="cuda")
                                  .view(torch.float8_e8m0fnu) for _ in range(2))
    c.tables = torch.full((sequences, width), -1, dtype=torch.int32, device="cuda")
    c.lengths = torch.zeros(sequences, dtype=torch.int32, device="cuda")
    c.slots = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
    return c


def _quantised_pages(case, seed, pages):
    """Pages of a cache that has been written: k, v and their scales."""
    out = []
    for x in _values(case, seed, pages):
        codes, scales = _quantise(x.float(), case["storage"], case["dtype"])
        out += [_elements(codes, case["storage"]), scales.transpose(-1, -2).contiguous().view(torch.float8_e8m0fnu)]
    return out[0], out[2], out[1], out[3]


def prepare(case, seed):
    kind, state = case["kind"], dict(case=case)
    dtype = DTYPES[case["dtype"]]
    if kind == "rope":
        q, k, v, positions, inv_freq, weights = _rope_inputs(case, seed)
        cache = None
        if case["store"] != "rows":
            slots, pages, _ = _slots(case, seed)
            cache = _cache(case, pages, pages, 1, case["N"], None if case["store"] == "pages" else case["store"])
            cache.slots.copy_(torch.tensor(slots, device="cuda"))
        if own:
            from llm_gpu_kernels_amd import prepare_qk_norm_rope
            more = dict(v=v, cache=cache, layer=0) if cache is not None else {}
            plan = prepare_qk_norm_rope(q, k, positions, inv_freq, *weights, eps=1e-6, interleaved=case["neighbours"], **more)
            return dict(state, plan=plan, cache=cache)
        return dict(state, q=q, k=k, v=v, positions=positions, inv_freq=inv_freq, weights=weights, cache=cache)
    if kind in ("append", "store"):
        k, v = _rows(case, _generator(seed), [case["Hkv"]] * 2)
        slots, pages, order = _slots(case, seed)
        cache = _cache(case, pages, pages, 1, case["N"], case["storage"])
        cache.slots.copy_(torch.tensor(slots, device="cuda"))
        state.update(cache=cache, k=k, v=v)
        if kind == "store":
            used = -(-case["N"] // case["page"])
            cache.tables.copy_(_int32([order[:used] + [-1] * (pages - used)]))
            cache.lengths.copy_(_int32([case["N"]]))
            state.update(rows=_int32([0]), starts=_int32([0, case["N"]]), k_out=torch.zeros(k.shape, dtype=dtype, device="cuda"),
                         v_out=torch.zeros(v.shape, dtype=dtype, device="cuda"))
        return state
    if kind == "read":
        lengths, pages, width, tables = _paged_inputs(case, seed)
        cache = _cache(case, pages, width, len(lengths), sum(lengths), case["storage"])
        for to, value in zip((cache.k, cache.v, cache.k_scales, cache.v_scales), _quantised_pages(case, seed, pages)):
            to.view(torch.uint8).copy_(value.view(torch.uint8)[None])
        cache.tables.copy_(_int32(tables))
        cache.lengths.copy_(_int32(lengths))
        k_out, v_out = (torch.zeros((sum(lengths), case["Hkv"], case["D"]), dtype=dtype, device="cuda") for _ in range(2))
        return dict(state, cache=cache, rows=_int32(range(len(lengths))), starts=_int32(_starts(lengths)), k_out=k_out,
                    v_out=v_out)
    if kind == "decode":
        lengths, pages, width, tables = _paged_inputs(case, seed)
        k, v, ks, vs = _quantised_pages(case, seed, pages)
        q = _randn((len(lengths), case["Hq"], case["D"]), _generator(int(seed) + 9), dtype, 1.5)
        tables, lengths = _int32(tables), _int32(lengths)
        if own:
            from llm_gpu_kernels_amd import prepare_paged_gqa
            return dict(state, plan=prepare_paged_gqa(q, k, v, tables, lengths, k_scales=ks, v_scales=vs))
        return dict(state, q=q, k=k, v=v, k_scales=ks, v_scales=vs, tables=tables, lengths=lengths)
    q, k, v, tables, lengths, members, prefixes = _shared_inputs(case, seed)
    tables, lengths, starts, prefixes = _int32(tables), _int32(lengths), _int32(_starts(members)), _int32(prefixes)
    if own:
        from llm_gpu_kernels_amd import prepare_shared_gqa
        return dict(state, plan=prepare_shared_gqa(q, k, v, tables, lengths, starts, prefixes))
    return dict(state, q=q, k=k, v=v, tables=tables, lengths=lengths, starts=starts, prefixes=prefixes,
                most=dict(members=max(members), prefix=max(_groups(case)[1])))


# ---- one pass -----------------------------------------------------------------


def _elements(codes, storage):
    return codes.view(torch.float8_e4m3fn if storage == "mxfp8" else torch.float4_e2m1fn_x2)


def _quantise(x, storage, dtype):
    """Rows [..., D] in 32 bits -> bytes of their elements [..., D or D / 2] and of
    their scales [..., D / 32]."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    top, last = LARGEST[storage]
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1))
    e = exponent - 1 - last + (2 * mantissa > top)
    e = e.clamp(FIRST_EXPONENT, LAST_EXPONENT[storage, dtype])
    inverse = ((127 - e) << 23).view(torch.float32)  # 2^-e (torch's own powers of two are not exact)
    y = (blocks * inverse[..., None]).clamp(-top * 2 ** last, top * 2 ** last).flatten(-2)
    scales = (e + 127).to(torch.uint8)
    if storage == "mxfp8":
        return y.to(torch.float8_e4m3fn).view(torch.uint8), scales
    a = y.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    code = code + 8 * (y < 0).to(torch.uint8)
    return code[..., 0::2] + 16 * code[..., 1::2], scales


def _dequantise(codes, scales, storage):
    """The values of rows of bytes [..., D or D / 2] with scales [..., D / 32]."""
    if storage == "mxfp8":
        x = codes.view(torch.float8_e4m3fn).float()
    else:
        values = torch.tensor(FP4 + tuple(-a for a in FP4), device="cuda")
        x = values[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()]
    return (x.unflatten(-1, (-1, BLOCK)) * scales.view(torch.float8_e8m0fnu).float()[..., None]).flatten(-2)


def _put(t, scales, slots, page, x, storage, dtype):
    """Rows [n, heads, D] in 32 bits to their slots of one layer, and their scales."""
    p, offset = slots // page, slots % page
    if storage is None:
        t[0][p, :, offset] = x.to(t.dtype)
        return
    codes, exponents = _quantise(x, storage, dtype)
    t.view(torch.uint8)[0][p, :, offset] = codes
    scales.view(torch.uint8)[0][p, :, :, offset] = exponents


def _get(t, scales, slots, page, storage, dtype):
    p, offset = slots // page, slots % page
    return _dequantise(t.view(torch.uint8)[0][p, :, offset], scales.view(torch.uint8)[0][p, :, :, offset], storage).to(dtype)


def _norm_rotate(x, weight, cos, sin, neighbours):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if neighbours:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_rope(s):
    case, c = s["case"], s["cache"]
    angles = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angles.cos().float(), angles.sin().float()
    q, k = (_norm_rotate(s[n], w, cos, sin, case["neighbours"]) for n, w in zip("qk", s["weights"]))
    q = q.to(DTYPES[case["dtype"]])
    if c is None:
        return q, k.to(q.dtype)
    storage = None if case["store"] == "pages" else case["store"]
    _put(c.k, getattr(c, "k_scales", None), c.slots, case["page"], k, storage, case["dtype"])
    _put(c.v, getattr(c, "v_scales", None), c.slots, case["page"], s["v"].float(), storage, case["dtype"])
    return q, None


def _written(c):
    return dict(k=c.k[0], v=c.v[0], **({} if getattr(c, "k_scales", None) is None
                                       else dict(k_scales=c.k_scales[0], v_scales=c.v_scales[0])))


def _plain_append(s):
    case, c = s["case"], s["cache"]
    _put(c.k, c.k_scales, c.slots, case["page"], s["k"].float(), case["storage"], case["dtype"])
    _put(c.v, c.v_scales, c.slots, case["page"], s["v"].float(), case["storage"], case["dtype"])


def _plain_gather(s):
    """Rows of the cache, one behind the other."""
    case, c, page = s["case"], s["cache"], s["case"]["page"]
    n, rows = s["k_out"].shape[0], s["rows"].long()
    counts = (s["starts"][1:] - s["starts"][:-1]).long()
    row = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts, output_size=n)
    j = torch.arange(n, device="cuda") - s["starts"].long()[row]
    slots = c.tables[rows[row], j // page].long() * page + j % page
    s["k_out"].copy_(_get(c.k, c.k_scales, slots, page, case["storage"], s["k_out"].dtype))
    s["v_out"].copy_(_get(c.v, c.v_scales, slots, page, case["storage"], s["v_out"].dtype))


def _softmax(scores):
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_decode(s):
    """Every sequence's keys and values side by side, as long as the longest."""
    case, q = s["case"], s["q"]
    kv, d, b = case["Hkv"], case["D"], q.shape[0]
    pages = s["tables"].clamp(min=0).long()

    def rows(t, scales):
        t, scales = t.view(torch.uint8)[pages], scales.view(torch.uint8)[pages]
        t = _dequantise(t, scales.transpose(-1, -2), case["storage"])
        return t.transpose(1, 2).reshape(b, kv, -1, d)

    k, v = rows(s["k"], s["k_scales"]), rows(s["v"], s["v_scales"])
    hidden = torch.arange(k.shape[2], device="cuda") >= s["lengths"][:, None]
    scores = torch.matmul(q.float().view(b, kv, -1, d), k.transpose(-1, -2)) / math.sqrt(d)
    p = _softmax(scores.masked_fill(hidden[:, None, None], -math.inf))
    return torch.matmul(p, v).view(q.shape).to(q.dtype)


def _plain_shared(s):
    """Prefixes once for each group, the rest for each sequence, one softmax."""
    case, q, page = s["case"], s["q"], s["case"]["page"]
    kv, d, b = case["Hkv"], case["D"], q.shape[0]
    groups, most, prefix = case["G"], s["most"]["members"], s["prefixes"].long()
    starts = s["starts"].long()
    member = torch.arange(b, device="cuda")
    g = torch.bucketize(member, starts[1:], right=True)
    place = member - starts[g]

    def grouped(x):  # [B, kv, group, n] -> [G, kv, most * group, n]
        t = torch.zeros((groups, most) + x.shape[1:], device="cuda")
        t[g, place] = x
        return t.transpose(1, 2).flatten(2, 3)

    def single(x):   # and back
        return x.unflatten(2, (most, -1)).transpose(1, 2)[g, place]

    first = s["tables"][starts[:-1], :-(-s["most"]["prefix"] // page)].clamp(min=0).long()
    kp, vp = (t[first].float().transpose(1, 2).reshape(groups, kv, -1, d) for t in (s["k"], s["v"]))
    qs = q.float().view(b, kv, -1, d)
    hidden = torch.arange(kp.shape[2], device="cuda") >= prefix[:, None]
    sp = torch.matmul(grouped(qs), kp.transpose(-1, -2)) / math.sqrt(d)
    sp = single(sp.masked_fill_(hidden[:, None, None], -math.inf))
    j = prefix[g][:, None] + torch.arange(case["tail"], device="cuda")
    seen = j < s["lengths"][:, None]
    pages = torch.gather(s["tables"], 1, (j // page).clamp(max=s["tables"].shape[1] - 1)).clamp(min=0).long()
    ks, vs = (t[pages, :, j % page].float().transpose(1, 2) for t in (s["k"], s["v"]))
    ss = torch.matmul(qs, ks.transpose(-1, -2)) / math.sqrt(d)
    ss = ss.masked_fill_(~seen[:, None, None], -math.inf)
    p = _softmax(torch.cat([sp, ss], -1))
    n = sp.shape[-1]
    out = single(torch.matmul(grouped(p[..., :n]), vp)) + torch.matmul(p[..., n:], vs)
    return out.reshape(q.shape).to(q.dtype)


def run(state):
    kind, c = state["case"]["kind"], state.get("cache")
    if kind == "rope":
        q, k = state["plan"].run() if own else _plain_rope(state)
        return dict(q=q, k=k) if c is None else dict(q=q, **_written(c))
    if kind in ("append", "store"):
        if own:
            c.append(0, state["k"], state["v"])
        else:
            _plain_append(state)
        if kind == "append":
            return _written(c)
    if kind in ("store", "read"):
        if own:
            c.gather(0, state["rows"], state["starts"], state["k_out"], state["v_out"])
        else:
            _plain_gather(state)
        return dict(k=state["k_out"], v=state["v_out"])
    if own:
        return state["plan"].run()
    return _plain_decode(state) if kind == "decode" else _plain_shared(state)


# ---- what a pass cannot do without ----------------------------------------------


def _row_bytes(case, storage):
    """Bytes of one token's keys or values."""
    d = case["D"]
    return case["Hkv"] * {None: 2 * d, "mxfp8": d + d // BLOCK, "mxfp4": d // 2 + d // BLOCK}[storage]


def work(case):
    kind, d = case["kind"], case["D"]
    if kind == "rope":
        n, rows = case["N"], case["Hq"] + case["Hkv"]
        store = None if case["store"] in ("rows", "pages") else case["store"]
        k = _row_bytes(case, None)
        moved = 2 * case["Hq"] * d * 2 + k + _row_bytes(case, store) + (0 if case["store"] == "rows" else
                                                                       k + _row_bytes(case, store) + 8)
        return dict(bytes=n * (moved + 4) + 2 * case["R"] + 4 * d * case["norm"],
                    flops=n * rows * (3 * case["R"] + 4 * d * case["norm"]))
    if kind in ("append", "store"):
        bits = _row_bytes(case, case["storage"])
        once = 2 * (_row_bytes(case, None) + bits)
        return dict(bytes=case["N"] * (once * (1 if kind == "append" else 2) + 8), flops=0)
    if kind == "read":
        n = sum(_lengths(case))
        return dict(bytes=n * 2 * (_row_bytes(case, None) + _row_bytes(case, case["storage"])), flops=0)
    q = 2 * case["Hq"] * d * 2
    if kind == "decode":
        lengths = _lengths(case)
        keys, pages = sum(lengths), sum(-(-n // case["page"]) for n in lengths)
        return dict(bytes=keys * 2 * _row_bytes(case, case["storage"]) + case["S"] * (q + 4) + 4 * pages,
                    flops=4 * case["Hq"] * d * keys)
    members, prefixes, lengths = _groups(case)
    owner = [g for g, n in enumerate(members) for _ in range(n)]
    keys = sum(prefixes) + sum(n - prefixes[g] for n, g in zip(lengths, owner))
    return dict(bytes=keys * 2 * _row_bytes(case, None) + len(lengths) * (q + 4) + 4 * (keys // case["page"]),
                flops=4 * case["Hq"] * d * sum(lengths))


# ---- the same in 64 bits ----------------------------------------------------------


def _exact_round(x, storage, dtype):
    """What 32 neighbours stand for once quantised, in 64 bits, and their scales."""
    x = x.double()
    blocks = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    bits, least, largest, top = {"mxfp8": (3, -6, 448.0, 8), "mxfp4": (1, 0, 6.0, 2)}[storage]

    def two(e):  # 2^e by its bits
        return (e.long() + 1023 << 52).view(torch.float64)

    most = blocks.abs().amax(-1)
    e = torch.frexp(most).exponent - 1 - top
    e = torch.where(most > largest * two(e), e + 1, e)
    scale = two(e.clamp(FIRST_EXPONENT, LAST_EXPONENT[storage, dtype]))
    y = blocks / scale[..., None]
    step = two((torch.frexp(y).exponent - 1).clamp(min=least) - bits)
    y = (torch.round(y / step) * step).clamp(-largest, largest)
    return y.reshape(x.shape), scale


def _exact_values(y, scale):
    return y * scale.repeat_interleave(32, dim=-1)


def _exact_put(shape, rows, slots, page):
    """[n, heads, m] to their places in zeros [pages, heads, page, m]."""
    out = torch.zeros(shape[0] * page, shape[1], rows.shape[-1], dtype=torch.float64, device="cuda")
    out[torch.tensor(slots, device="cuda")] = rows
    return out.view(shape[0], page, shape[1], rows.shape[-1]).permute(0, 2, 1, 3)


def _exact_pages(x, case, slots, pages, storage):
    """Elements and scales of a layer in which rows x [n, heads, D] were written."""
    shape, page = (pages, case["Hkv"]), case["page"]
    if storage is None:
        return _exact_put(shape, x.double(), slots, page), None
    y, scale = _exact_round(x, storage, case["dtype"])
    scales = _exact_put(shape, scale, slots, page).transpose(-1, -2)
    return _exact_put(shape, y, slots, page), torch.where(scales == 0, 2.0 ** -127, scales)


def _exact_rope(case, seed):
    q, k, v, positions, inv_freq, weights = _rope_inputs(case, seed)
    half = case["R"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       positions.double()[:, None, None] * inv_freq.double())

    def one(x, weight):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["D"] + 1e-6) * weight.double()
        pairs = [2 * i for i in range(half)] if case["neighbours"] else list(range(half))
        a = torch.tensor(pairs, device="cuda")
        b = a + (1 if case["neighbours"] else half)
        z = torch.complex(x[..., a], x[..., b]) * turn
        x = x.clone()
        x[..., a], x[..., b] = z.real, z.imag
        return x

    q, k = one(q, weights[0]), one(k, weights[1])
    if case["store"] == "rows":
        return dict(q=q, k=k)
    slots, pages, _ = _slots(case, seed)
    storage = None if case["store"] == "pages" else case["store"]
    (k, ks), (v, vs) = (_exact_pages(x, case, slots, pages, storage) for x in (k, v))
    return dict(q=q, k=k, v=v, **({} if storage is None else dict(k_scales=ks, v_scales=vs)))


def _exact_head(q, k, v):
    """softmax(q k^T / sqrt(D)) v of one sequence and key head in 64 bits."""
    s = torch.mm(q, k.t()) * q.shape[-1] ** -0.5
    return torch.mm(torch.softmax(s, -1), v)


def exact(case, seed):
    kind = case["kind"]
    if kind == "rope":
        return _exact_rope(case, seed)
    if kind in ("append", "store"):
        k, v = _rows(case, _generator(seed), [case["Hkv"]] * 2)
        if kind == "store":
            return dict(zip("kv", (_exact_values(*_exact_round(x, case["storage"], case["dtype"])) for x in (k, v))))
        slots, pages, _ = _slots(case, seed)
        (k, ks), (v, vs) = (_exact_pages(x, case, slots, pages, case["storage"]) for x in (k, v))
        return dict(k=k, v=v, k_scales=ks, v_scales=vs)
    group, page = case["Hq"] // case["Hkv"] if "Hq" in case else 0, case["page"]
    if kind in ("read", "decode"):
        lengths, pages, _, tables = _paged_inputs(case, seed)
        k, v = (_exact_values(*_exact_round(x, case["storage"], case["dtype"])) for x in _values(case, seed, pages))
        if kind == "decode":
            q = _randn((len(lengths), case["Hq"], case["D"]), _generator(int(seed) + 9), DTYPES[case["dtype"]], 1.5)
    else:
        q, k, v, tables, lengths, _, _ = _shared_inputs(case, seed)
    out = []
    for b, n in enumerate(lengths):
        used = torch.tensor(tables[b][:-(-n // page)], device="cuda")
        kb, vb = (t[used].double().permute(1, 0, 2, 3).reshape(case["Hkv"], -1, case["D"])[:, :n] for t in (k, v))
        if kind == "read":
            out.append((kb.transpose(0, 1), vb.transpose(0, 1)))
            continue
        qb = q[b].double().view(case["Hkv"], group, -1)
        out.append(torch.cat([_exact_head(qb[h], kb[h], vb[h]) for h in range(case["Hkv"])]))
    if kind == "read":
        return dict(k=torch.cat([x for x, _ in out]), v=torch.cat([x for _, x in out]))
    return torch.stack(out)
