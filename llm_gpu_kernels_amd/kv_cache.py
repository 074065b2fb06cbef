"""Paged key-value cache on MI355X (no counterpart in the reference).

``PagedKVCache`` owns the keys and values of every layer in pages, and the whole
bookkeeping (page tables, lengths, holders of each page) on the GPU.  A serving
step enqueues ``reserve`` (room for new tokens), one ``append`` per layer (their
keys and values) and attention (``prepare_packed_gqa`` for whole prompts,
``prepare_paged_gqa`` for single tokens); ``fork`` and ``free`` start and end
sequences that share pages, ``compact`` moves the pages in use to the front.
No method synchronises or allocates, so all of them can be captured in a HIP
graph; calls on one cache must run in stream order.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from .attention import _check_int32, _stream_of

__all__ = ["PagedKVCache"]


class PagedKVCache:
    """Keys and values of up to ``sequences`` rows in ``pages`` pages.

    Attributes (tensors on the GPU, updated in place):

    * ``k``, ``v`` [layers, pages, kv_heads, page_size, head_dim];
    * ``tables`` int32 [sequences, max_pages]: each row's pages, -1 behind them;
    * ``lengths`` int32 [sequences]: tokens of each row, 0 if it is empty;
    * ``refs`` int32 [pages]: rows that hold the page, 0 if it is free;
    * ``slots`` int64 [max_tokens]: where the tokens of the last ``reserve`` go
      (page * page_size + row in the page), -1 for none;
    * ``starts`` int32 [sequences + 1]: running sums of the last ``reserve``'s
      counts, as ``prepare_packed_gqa`` takes them;
    * ``used_pages`` int32 [1]: pages in use at the last ``compact``.

    Values that a call on the GPU cannot serve are left out and latch a status
    (``read_status``, ``check_inputs``).
    """

    def __init__(self, pages, page_size, kv_heads, head_dim, *, sequences, max_pages, max_tokens, layers=1,
                 dtype=torch.bfloat16, device="cuda"):
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("dtype must be torch.bfloat16 or torch.float16")
        device = torch.device(device)
        d = N.KvCacheDesc()
        sizes = dict(pages=pages, page_size=page_size, kv_heads=kv_heads, head_dim=head_dim, layers=layers,
                     sequences=sequences, max_pages=max_pages, max_tokens=max_tokens)
        for name, value in sizes.items():
            if not isinstance(value, int) or isinstance(value, bool) or not -2 ** 31 <= value < 2 ** 31:
                raise ValueError(f"{name} must be an int (got {value!r})")
            setattr(d, name, value)
        nbytes, handle = ctypes.c_size_t(0), ctypes.c_void_p()
        N.check(N.lib().kv_cache_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)), "cache")
        if device.type != "cuda":
            raise ValueError("device must be a GPU device")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, kv_heads, head_dim
        self.sequences, self.max_pages, self.max_tokens, self.layers = sequences, max_pages, max_tokens, layers
        self.dtype, self.device = dtype, device
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)

        def ints(*size, value=0, kind=torch.int32):
            return torch.full(size, value, dtype=kind, device=device)

        self.tables, self.lengths, self.refs = ints(sequences, max_pages, value=-1), ints(sequences), ints(pages)
        self.slots, self.starts = ints(max_tokens, value=-1, kind=torch.int64), ints(sequences + 1)
        self._status = ints(4)
        self.used_pages = self._status[1:2]
        self.workspace = torch.zeros(int(nbytes.value), dtype=torch.uint8, device=device)
        for name in ("k", "v", "tables", "lengths", "refs", "starts", "slots", "workspace"):
            setattr(d, name, getattr(self, name).data_ptr())
        d.status, d.workspace_bytes = self._status.data_ptr(), self.workspace.numel()
        with torch.cuda.device(device):
            N.check(N.lib().kv_cache_create(ctypes.byref(handle), ctypes.byref(d)), "cache")
        self._desc, self._cache = d, handle

    def _stream(self):
        return _stream_of(self.device)

    def _token_stride(self, t, name):
        """Token stride of new keys or values (alignment is checked by the library)."""
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        heads, dim = self.kv_heads, self.head_dim
        shape = t.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != dim or t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"{name} must be {self.dtype} [n, {heads}, {dim}] on {self.device}")
        s0, s1, s2 = t.stride()
        if shape[0] == 0:
            return heads * dim
        if s2 != 1 or (heads > 1 and s1 != dim):
            raise ValueError(f"{name} must have inner strides ({dim}, 1)")
        return s0 if shape[0] > 1 else heads * dim

    def _rows(self, t, name):
        if not isinstance(t, torch.Tensor) or t.ndim != 1:
            raise ValueError(f"{name} must be an int32 tensor [n]")
        _check_int32(t, name, (t.shape[0],), self.device)
        if t.shape[0] > self.sequences:
            raise ValueError(f"{name} must name at most {self.sequences} rows (got {t.shape[0]})")
        return t

    def reserve(self, counts, stride=0):
        """Room for ``counts[s]`` more tokens in every row s (int32 [sequences]).

        Sets ``slots`` and ``starts``: with ``stride`` 0 the tokens lie packed,
        those of row s from ``starts[s]`` on; with a stride n those of row s from
        ``s * n`` on (a decode step with one place per row: 1).  Pages are handed
        out lowest number first to the rows in order; a partly filled last page
        that other rows hold too is copied first (where all its holders grow in
        one call, the last of them keeps the page).  All or nothing: a call that
        cannot be served changes no row and sets all slots to -1."""
        _check_int32(counts, "counts", (self.sequences,), self.device)
        if not isinstance(stride, int) or stride < 0 or stride * self.sequences > self.max_tokens:
            raise ValueError(f"stride must be an int >= 0, stride * sequences at most {self.max_tokens}")
        N.check(N.lib().kv_cache_reserve(self._cache, counts.data_ptr(), stride, self._stream()), "reserve")

    def append(self, layer, k, v):
        """Write token i's keys and values ([n, kv_heads, head_dim], the heads of
        a token side by side) to ``slots[i]`` of a layer, for every i < n whose
        slot is not -1."""
        if not isinstance(layer, int) or not 0 <= layer < self.layers:
            raise ValueError(f"layer must be an int in [0, {self.layers}) (got {layer!r})")
        ks, vs = self._token_stride(k, "k"), self._token_stride(v, "v")
        if k.shape[0] != v.shape[0]:
            raise ValueError("k and v must have the same number of tokens")
        N.check(N.lib().kv_cache_append(self._cache, layer, k.data_ptr(), v.data_ptr(), ks, vs, k.shape[0],
                                        self._stream()), "append")

    def fork(self, src, dst):
        """Row ``dst[i]``, which must be empty, starts as a copy of row ``src[i]``
        that shares its pages (int32 [n]; a pair with a negative row is left
        out).  All rows are read as they are before the call."""
        src, dst = self._rows(src, "src"), self._rows(dst, "dst")
        if src.shape != dst.shape:
            raise ValueError("src and dst must have the same length")
        N.check(N.lib().kv_cache_fork(self._cache, src.data_ptr(), dst.data_ptr(), src.shape[0], self._stream()), "fork")

    def free(self, rows):
        """Empty the rows (int32 [n]; negative ones are left out).  Pages that no
        row holds any more are free."""
        rows = self._rows(rows, "rows")
        N.check(N.lib().kv_cache_free(self._cache, rows.data_ptr(), rows.shape[0], self._stream()), "free")

    def compact(self):
        """Move the pages in use to the front, in every layer, and the tables
        with them: with U pages in use (``used_pages``) the i-th free page below
        U takes the i-th used page from U on."""
        N.check(N.lib().kv_cache_compact(self._cache, self._stream()), "compact")

    def read_status(self) -> int:
        """Synchronise; the status bits of the calls since the last reading."""
        flags = ctypes.c_uint32(0)
        N.check(N.lib().kv_cache_read_status(self._cache, self._stream(), ctypes.byref(flags)), "status")
        return int(flags.value)

    def check_inputs(self):
        """Synchronising check of the calls since the last one."""
        flags = self.read_status()
        if flags & (N.KV_STATUS_OUT_OF_PAGES | N.KV_STATUS_TOO_LONG):
            raise RuntimeError(f"the cache has no room for a reserve: GPU status={flags} "
                               "(4=free pages, 8=max_pages of a row)")
        if flags:
            raise ValueError(f"invalid runtime cache inputs: GPU status={flags} (1=rows, 2=fork destinations, "
                             "16=counts, 32=lengths or page numbers)")

    def __del__(self):
        cache = getattr(self, "_cache", None)
        if cache is not None and cache.value:
            try:
                N.lib().kv_cache_destroy(cache)
            except Exception:
                pass
            self._cache = None
