"""Norms of queries and keys for each head and their rotation by position on MI355X,
in one pass, with the keys and values written to a cache on the way (no counterpart in
the reference).

``prepare_qk_norm_rope`` has the form and lifetime of the attention plans: it binds its
tensors by address, ``run()`` enqueues on the current stream without a host sync or an
allocation, and can be captured in a HIP graph.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _native as N
from .attention import _DTYPES, _check_int32, _check_rows, _output, _set_sizes, _stream_of, _token_stride, check_out_storage
from .kv_cache import PagedKVCache

__all__ = ["PreparedQKNormRope", "prepare_qk_norm_rope"]


def _check_vector(t, name, size, dtypes, device):
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise TypeError(f"{name} must be a tensor of {' or '.join(map(str, dtypes))}")
    if t.ndim != 1 or (size is not None and t.shape[0] != size):
        raise ValueError(f"{name} must have shape [{'n' if size is None else size}], got {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if t.shape[0] > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")


def _span(t):
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


class PreparedQKNormRope:
    """Owns the outputs; binds everything else by address, and keeps the cache."""

    def __init__(self, q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, q_out=None,
                 k_out=None, v=None, cache=None, layer=0):
        _check_rows(q, "q")
        _check_rows(k, "k", like=q)
        if k.shape[0] != q.shape[0]:
            raise ValueError("k must have q's number of tokens")
        device, (n, hq, dim), hkv = q.device, q.shape, k.shape[1]
        _check_int32(positions, "positions", (n,), device)
        _check_vector(inv_freq, "inv_freq", None, (torch.float32,), device)
        if not 1 <= inv_freq.shape[0] <= dim // 2:
            raise ValueError(f"inv_freq must have 1 to {dim // 2} entries (got {inv_freq.shape[0]})")
        weights = [t for t in (q_weight, k_weight) if t is not None]
        for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
            if t is not None:
                _check_vector(t, name, dim, (q.dtype, torch.float32), device)
        if len(weights) == 2 and weights[0].dtype != weights[1].dtype:
            raise TypeError("q_weight and k_weight must have one dtype")
        if not (math.isfinite(float(eps)) and 0.0 <= float(eps) <= 3e38):
            raise ValueError(f"eps must be finite and not negative (got {eps!r})")
        if (v is None) != (cache is None):
            raise ValueError("v and cache must be given together")
        if cache is not None:
            if not isinstance(cache, PagedKVCache):
                raise TypeError("cache must be a PagedKVCache")
            _check_rows(v, "v", like=q)
            if v.shape != k.shape:
                raise ValueError("v must have k's shape")
            if cache.dtype != q.dtype or cache.device != device:
                raise ValueError("cache must have q's dtype and device")
            if not isinstance(layer, int) or not 0 <= layer < cache.layers:
                raise ValueError(f"layer must be an int in [0, {cache.layers}) (got {layer!r})")
        if device.type != "cuda":
            raise ValueError("q must be on a GPU device")
        d = N.QkNormRopeDesc()
        _set_sizes(d, N=n, Hq=hq, Hkv=hkv, D=dim, R=2 * inv_freq.shape[0], dtype=_DTYPES[q.dtype], layer=0 if cache is None else layer)
        d.interleaved, d.weights_fp32 = bool(interleaved), bool(weights and weights[0].dtype == torch.float32)
        d.q_stride, d.k_stride, d.eps = _token_stride(q, "q"), _token_stride(k, "k"), float(eps)
        d.v_stride = 0 if v is None else _token_stride(v, "v")
        q_out = _output(q_out, q)
        k_out = None if k_out is None and cache is not None else _output(k_out, k)
        inputs = [q, k, positions, inv_freq] + weights
        if cache is not None:
            inputs += [v, cache.k, cache.v, cache.slots] + [t for t in (cache.k_scales, cache.v_scales) if t is not None]
        for out in (q_out, k_out):
            if out is not None:
                check_out_storage(out, inputs)
        if k_out is not None and k_out.numel():
            (a, b), (c, e) = _span(q_out), _span(k_out)
            if a < e and c < b:
                raise ValueError("q_out and k_out must not overlap")
        self.q, self.k, self.v, self.positions, self.inv_freq = q, k, v, positions, inv_freq
        self.q_weight, self.k_weight, self.cache, self.q_out, self.k_out = q_weight, k_weight, cache, q_out, k_out
        for name in ("q", "k", "v", "positions", "inv_freq", "q_weight", "k_weight", "q_out", "k_out"):
            t = getattr(self, name)
            setattr(d, name, None if t is None else t.data_ptr())
        handle = ctypes.c_void_p()
        with torch.cuda.device(device):
            N.check(N.lib().qk_norm_rope_create(ctypes.byref(handle), ctypes.byref(d), None if cache is None else cache._cache),
                    "prepare")
        self._plan, self._device, self._run = handle, device, N.lib().qk_norm_rope_run

    def run(self):
        """Enqueue one pass on the current stream; returns (q_out, k_out)."""
        N.check(self._run(self._plan, _stream_of(self._device)), "run")
        return self.q_out, self.k_out

    def __del__(self):
        plan = getattr(self, "_plan", None)
        if plan is not None and plan.value:
            try:
                N.lib().qk_norm_rope_destroy(plan)
            except Exception:
                pass
            self._plan = None


def prepare_qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, *, eps=1e-6, interleaved=False, q_out=None,
                         k_out=None, v=None, cache=None, layer=0):
    """Norm and rotate the queries and keys of N tokens, and cache keys and values.

    ``q`` [N, Hq, D] and ``k`` [N, Hkv, D], bf16 or fp16, D 64 or 128, the heads of a
    token side by side (views of one fused projection will do).  For every head x:
    ``y = x * weight / sqrt(mean(x^2) + eps)`` with ``q_weight`` or ``k_weight`` ([D], of
    q's dtype or float32; None: ``y = x``), and for i < R/2 = ``len(inv_freq)`` the
    elements i and i + R/2 (2 i and 2 i + 1 with ``interleaved``) turn by the angle
    ``positions[t] * inv_freq[i]``; elements from R on stay.  ``positions`` int32 [N],
    ``inv_freq`` float32.  In fp32 (angles in 64 bits), rounded once.

    With ``v`` [N, Hkv, D] and a ``cache``, token t's keys, so treated, and its values
    go to ``cache.slots[t]`` of ``layer`` (-1: nowhere), as ``append`` writes them;
    a cache with a storage quantises the keys from fp32.  ``run()`` returns
    ``(q_out, k_out)``; with a cache k_out is None unless it is given.  Values of all
    tensors may change in place between runs.  Prepares and runs once."""
    plan = PreparedQKNormRope(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved, q_out, k_out, v, cache, layer)
    plan.run()
    return plan
