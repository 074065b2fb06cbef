"""Segmented-KV GQA prefill attention on MI355X (secondary path).

Mirrors ``prepare_cuda_gqa_compact(q, segments, out=None, *, stages=1)``
(src/llm_gpu_kernels/attention_cuda_compact.py:135-186) and its input
validation (:97-121): Q [T, 32, 128] bf16 contiguous, segments = sequence of
(k, v) pairs [L, 8, 128] bf16 with inner strides (128, 1) and a token stride
>= heads*128 that is a multiple of 8, the last segment being the current
chunk (L == T, causal).  ``run()`` enqueues on the current stream with no
host sync and no allocation and returns the owned output.

``prepare_packed_gqa`` (several prompts in one call) and ``prepare_paged_gqa``
(one new token per sequence over the pages of a ``PagedKVCache``) have the same
form and lifetime; they have no counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _native as N

__all__ = ["PreparedSegmentedGQA", "prepare_segmented_gqa", "prepare_cuda_gqa_compact", "PreparedPackedGQA",
           "prepare_packed_gqa", "PreparedPagedGQA", "prepare_paged_gqa"]


def _validate(t, name, device, heads):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.ndim != 3 or tuple(t.shape[1:]) != (heads, 128):
        raise ValueError(f"{name} must have shape [L, {heads}, 128]")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must have dtype torch.bfloat16")
    if t.device != device:
        raise ValueError(f"{name} must be on q's device")
    if tuple(t.stride()[1:]) != (128, 1):
        raise ValueError(f"{name} must have inner strides (128, 1)")
    if t.shape[0] and (t.stride(0) < heads * 128 or t.stride(0) % 8):
        raise ValueError(f"{name} token stride must be at least {heads * 128} and divisible by 8")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} base address must be 16-byte aligned")


def check_out_storage(out, inputs):
    """Reject an output that shares storage with q or a K/V segment: the kernel
    writes out while other workgroups still read the inputs
    (attention_cuda_compact.py:175-177 rejects the same).  Empty tensors own no
    memory and cannot alias."""
    if out.numel() == 0:
        return
    storage = out.untyped_storage().data_ptr()
    if any(t.numel() and t.untyped_storage().data_ptr() == storage for t in inputs):
        raise ValueError("out must not share storage with any input")


class PreparedSegmentedGQA:
    """Owns the output and split-K workspace; binds q and the segments by address."""

    def __init__(self, q, segments, out=None, scale=None):
        if not isinstance(q, torch.Tensor) or q.ndim != 3 or q.shape[2] != 128:
            raise ValueError("q must be [T, Hq, 128]")
        if scale is not None and not (math.isfinite(float(scale)) and float(scale) > 0.0):
            # the C ABI reads a scale <= 0 or non-finite as "default"; an explicit
            # one must not be replaced silently
            raise ValueError(f"scale must be a positive finite number (got {scale!r})")
        if q.dtype != torch.bfloat16 or not q.is_contiguous() or q.device.type != "cuda":
            raise ValueError("q must be a contiguous bf16 GPU tensor")
        segments = [tuple(s) for s in segments]
        if not 1 <= len(segments) <= N.GQA_MAX_SEGMENTS:
            raise ValueError("1..4 KV segments required")
        t, hq, _ = q.shape
        hkv = segments[0][0].shape[1]
        for i, (k, v) in enumerate(segments):
            _validate(k, f"segments[{i}].k", q.device, hkv)
            _validate(v, f"segments[{i}].v", q.device, hkv)
            if k.shape[0] != v.shape[0]:
                raise ValueError(f"segments[{i}] k and v lengths differ")
        if segments[-1][0].shape[0] != t:
            raise ValueError("the current (last) segment must have T tokens")
        if out is None:
            out = torch.empty_like(q)
        if tuple(out.shape) != tuple(q.shape) or out.dtype != torch.bfloat16 or not out.is_contiguous():
            raise ValueError("out must be a contiguous bf16 tensor shaped like q")
        check_out_storage(out, [q] + [t for pair in segments for t in pair])
        self.q, self.segments, self.output = q, segments, out
        d = N.GqaDesc()
        d.T, d.Hq, d.Hkv, d.D, d.num_segments = t, hq, hkv, 128, len(segments)
        for i, (k, v) in enumerate(segments):
            d.len[i] = k.shape[0]
            d.k[i] = k.data_ptr() if k.shape[0] else None
            d.v[i] = v.data_ptr() if v.shape[0] else None
            d.k_stride[i] = k.stride(0) if k.shape[0] else hkv * 128
            d.v_stride[i] = v.stride(0) if v.shape[0] else hkv * 128
        d.q, d.out = q.data_ptr(), out.data_ptr()
        d.scale = float(scale) if scale is not None else 1.0 / math.sqrt(128.0)
        nbytes = ctypes.c_size_t(0)
        with torch.cuda.device(q.device):
            N.check(N.lib().gqa_seg_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)), "prepare")
            self.workspace = torch.empty(max(int(nbytes.value), 16), dtype=torch.uint8, device=q.device)
            d.workspace, d.workspace_bytes = self.workspace.data_ptr(), self.workspace.numel()
            handle = ctypes.c_void_p()
            N.check(N.lib().gqa_seg_plan_create(ctypes.byref(handle), ctypes.byref(d)), "prepare")
        self._desc, self._plan = d, handle
        self.splits_workspace_bytes = int(nbytes.value)

    def run(self):
        if self.q.shape[0] == 0:
            return self.output
        stream = torch.cuda.current_stream(self.q.device).cuda_stream
        N.check(N.lib().gqa_seg_plan_run(self._plan, ctypes.c_void_p(stream)), "run")
        return self.output

    def __del__(self):
        plan = getattr(self, "_plan", None)
        if plan is not None and plan.value:
            try:
                N.lib().gqa_seg_plan_destroy(plan)
            except Exception:
                pass
            self._plan = None


def prepare_segmented_gqa(q, segments, out=None, *, scale=None):
    plan = PreparedSegmentedGQA(q, segments, out, scale)
    plan.run()
    return plan


def prepare_cuda_gqa_compact(q, segments, out=None, *, stages=1):
    """Reference entry point (attention_cuda_compact.py:135); ``stages`` is
    accepted for compatibility -- the gfx950 kernel's pipeline is fixed."""
    if stages not in (1, 2):
        raise ValueError("stages must be 1 or 2")
    return prepare_segmented_gqa(q, segments, out)


# ---- several prompts in one call, and one new token over a paged cache -----------

_DTYPES = {torch.bfloat16: N.GQA_BF16, torch.float16: N.GQA_FP16}


def _check_rows(t, name, ndim=3, like=None):
    """A [.., rows, heads or row, D] operand of the packed and paged calls."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.ndim != ndim or t.shape[-1] not in (64, 128):
        raise ValueError(f"{name} must have {ndim} dimensions, the last of 64 or 128")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must have dtype torch.bfloat16 or torch.float16")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[-1] != like.shape[-1]):
        raise ValueError(f"{name} must have q's dtype, device and head dimension")
    if t.numel() and t.stride(-1) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    if t.numel() and t.data_ptr() % 16:
        raise ValueError(f"{name} base address must be 16-byte aligned")


def _stride(t, dim, default):
    """The stride of a dimension; any will do for one that has a single entry."""
    return t.stride(dim) if t.numel() and t.shape[dim] > 1 else default


def _token_stride(t, name):
    """Token stride of [tokens, heads, D] with the heads of a token side by side."""
    heads, d = t.shape[1:]
    if _stride(t, 1, d) != d:
        raise ValueError(f"{name} must have inner strides ({d}, 1)")
    return _stride(t, 0, heads * d)


def _check_int32(t, name, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 tensor")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")


def _check_scale(scale, d):
    # The C ABI reads a scale <= 0 or non-finite as "default"; an explicit one
    # must not be replaced silently.
    if scale is None:
        return 1.0 / math.sqrt(d)
    if not (math.isfinite(float(scale)) and float(scale) > 0.0):
        raise ValueError(f"scale must be a positive finite number (got {scale!r})")
    return float(scale)


def _set_sizes(desc, **sizes):
    """32-bit fields of a descriptor (ctypes would drop the upper bits silently)."""
    for name, value in sizes.items():
        if value >= 2 ** 31:
            raise ValueError(f"{name} must be below 2^31 (got {value})")
        setattr(desc, name, value)


def _fp32_scale(scale, d):
    """The scale as the kernels use it: a normal fp32 number whose product with
    log2(e) is one too."""
    value = ctypes.c_float(_check_scale(scale, d)).value
    if not 2.0 ** -126 <= value <= 2.0 ** 127:
        raise ValueError(f"scale must lie in [2^-126, 2^127] (got {scale!r})")
    return value


# torch.cuda.current_stream() makes an object for every call: 1.1 us of the 5 that the
# host takes for one, so the stream's address is asked for directly where torch has that.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_of(device):
    """Address of the current stream of a device with a number."""
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


class _PreparedPlan:
    """A plan of the library with its workspace; ``run()`` enqueues on the
    current stream of q's device.  Runs of one plan must be in stream order."""

    _prefix = ""

    def _create(self, desc, device):
        fn = {n: getattr(N.lib(), f"{self._prefix}_{n}") for n in
              ("workspace_bytes", "plan_create", "plan_run", "plan_read_status", "plan_destroy")}
        nbytes, handle = ctypes.c_size_t(0), ctypes.c_void_p()
        if device.type != "cuda":
            raise ValueError("q must be on a GPU device")
        with torch.cuda.device(device):
            N.check(fn["workspace_bytes"](ctypes.byref(desc), ctypes.byref(nbytes)), "prepare")
            self.workspace = torch.zeros(int(nbytes.value), dtype=torch.uint8, device=device)
            desc.workspace, desc.workspace_bytes = self.workspace.data_ptr(), self.workspace.numel()
            N.check(fn["plan_create"](ctypes.byref(handle), ctypes.byref(desc)), "prepare")
        self._fn, self._run, self._desc, self._plan, self._device = fn, fn["plan_run"], desc, handle, device

    def run(self):
        """Enqueue one pass on the current stream; returns the owned output."""
        N.check(self._run(self._plan, _stream_of(self._device)), "run")
        return self.output

    def read_status(self) -> int:
        """Synchronise; the status bits of the passes since the last reading."""
        flags = ctypes.c_uint32(0)
        N.check(self._fn["plan_read_status"](self._plan, _stream_of(self._device), ctypes.byref(flags)), "status")
        return int(flags.value)

    def check_inputs(self):
        """Synchronising debug check of the passes since the last one."""
        flags = self.read_status()
        if flags:
            raise ValueError(f"invalid runtime attention inputs: GPU status={flags} "
                             "(1=starts or lengths, 2=page numbers)")

    def __del__(self):
        plan = getattr(self, "_plan", None)
        if plan is not None and plan.value:
            try:
                self._fn["plan_destroy"](plan)
            except Exception:
                pass
            self._plan = None


def _output(out, q):
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if not isinstance(out, torch.Tensor):
        raise TypeError("out must be a torch.Tensor")
    if tuple(out.shape) != tuple(q.shape) or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape, dtype and device")
    if out.numel() and out.data_ptr() % 16:
        raise ValueError("out base address must be 16-byte aligned")
    return out


class PreparedPackedGQA(_PreparedPlan):
    """Owns the output and workspace; binds q, k, v and starts by address."""

    _prefix = "gqa_packed"

    def __init__(self, q, k, v, starts, out=None, scale=None):
        _check_rows(q, "q")
        _check_rows(k, "k", like=q)
        _check_rows(v, "v", like=q)
        if k.shape != v.shape or k.shape[0] != q.shape[0]:
            raise ValueError("k and v must have one shape, with q's number of tokens")
        if not isinstance(starts, torch.Tensor) or starts.ndim != 1 or starts.shape[0] < 1:
            raise ValueError("starts must be an int32 tensor [sequences + 1]")
        _check_int32(starts, "starts", (starts.shape[0],), q.device)
        d = N.GqaPackedDesc()
        _set_sizes(d, N=q.shape[0], Hq=q.shape[1], D=q.shape[2], S=starts.shape[0] - 1, Hkv=k.shape[1],
                   dtype=_DTYPES[q.dtype])
        d.scale = _fp32_scale(scale, d.D)
        d.q_stride, d.k_stride, d.v_stride = (_token_stride(t, n) for t, n in ((q, "q"), (k, "k"), (v, "v")))
        out = _output(out, q)
        check_out_storage(out, [q, k, v, starts])
        self.q, self.k, self.v, self.starts, self.output = q, k, v, starts, out
        d.q, d.k, d.v, d.out, d.starts = (t.data_ptr() for t in (q, k, v, out, starts))
        self._create(d, q.device)


def prepare_packed_gqa(q, k, v, starts, out=None, *, scale=None):
    """Causal attention of several prompts packed behind each other.

    ``q`` [N, Hq, D], ``k`` and ``v`` [N, Hkv, D], bf16 or fp16, D 64 or 128, Hq
    a multiple of Hkv, the heads of a token side by side (views of one fused
    projection will do); ``starts`` int32 [S + 1] on the GPU: sequence s holds
    the tokens ``starts[s]`` to ``starts[s + 1] - 1``, none if they are equal.
    Values of all of them may change in place between runs.  Rows of ``output``
    that belong to no sequence keep what they held.  Prepares and runs once;
    ``run()`` has no host sync and no allocation."""
    plan = PreparedPackedGQA(q, k, v, starts, out, scale)
    plan.run()
    return plan


class PreparedPagedGQA(_PreparedPlan):
    """Owns the output and workspace; binds q, the pages, tables and lengths by
    address."""

    _prefix = "gqa_paged"

    def __init__(self, q, k_pages, v_pages, tables, lengths, out=None, scale=None):
        _check_rows(q, "q")
        _check_rows(k_pages, "k_pages", 4, q)
        _check_rows(v_pages, "v_pages", 4, q)
        if k_pages.shape != v_pages.shape:
            raise ValueError("k_pages and v_pages must have one shape")
        if not isinstance(tables, torch.Tensor) or tables.ndim != 2:
            raise ValueError("tables must be an int32 tensor [B, pages per sequence]")
        b, m = q.shape[0], tables.shape[1]
        _check_int32(tables, "tables", (b, m), q.device)
        _check_int32(lengths, "lengths", (b,), q.device)
        p, hkv, page, dim = k_pages.shape
        d = N.GqaPagedDesc()
        _set_sizes(d, B=b, Hq=q.shape[1], D=dim, Hkv=hkv, P=p, page=page, M=m, dtype=_DTYPES[q.dtype])
        d.scale = _fp32_scale(scale, dim)
        d.q_stride, d.table_stride = _token_stride(q, "q"), _stride(tables, 0, m)
        for t, into in ((k_pages, d.k_strides), (v_pages, d.v_strides)):
            into[0], into[1], into[2] = _stride(t, 0, 8), _stride(t, 1, 8), _stride(t, 2, dim)
        out = _output(out, q)
        check_out_storage(out, [q, k_pages, v_pages, tables, lengths])
        self.q, self.k_pages, self.v_pages, self.tables, self.lengths, self.output = (q, k_pages, v_pages, tables,
                                                                                      lengths, out)
        d.q, d.k, d.v, d.out, d.tables, d.lengths = (t.data_ptr() for t in (q, k_pages, v_pages, out, tables, lengths))
        self._create(d, q.device)


def prepare_paged_gqa(q, k_pages, v_pages, tables, lengths, out=None, *, scale=None):
    """Attention of one new token of each of B sequences over a paged cache.

    ``q`` [B, Hq, D], bf16 or fp16, D 64 or 128; ``k_pages`` and ``v_pages``
    [P, Hkv, page, D] of the same type (``cache.k[layer]``; other orders of the
    outer dimensions as permuted views), page a multiple of 16; ``tables`` int32
    [B, M] and ``lengths`` int32 [B] on the GPU: key j of sequence b is row
    ``j % page`` of page ``tables[b, j // page]``, and all ``lengths[b]`` keys
    are seen, the new token's own among them (``append`` it first).  Length 0
    gives zeros.  Values of all of them may change in place between runs; table
    entries behind a sequence's last page are not read.  Prepares and runs once;
    ``run()`` has no host sync and no allocation."""
    plan = PreparedPagedGQA(q, k_pages, v_pages, tables, lengths, out, scale)
    plan.run()
    return plan
