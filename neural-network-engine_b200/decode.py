"""The rest of a decode step around the linear layers: the paged key/value cache, the step that fills it, the attention
that reads it, and the draw of the next token.  Like the plans of ``quantized``, a call is set up once over device buffers
that stay in place and then run, on any stream, as often as the buffers hold something new.  Every
computation is a call through the ``nne_cuda`` C ABI; pointers are device addresses (0: not given).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np

from . import _lib
from ._lib import NneError, check, load
from .quantized import CudaContext, GpuError, InvalidArgument, _ptr, _raise_mapped

_DTYPES = {"f16": _lib.F16, "bf16": _lib.BF16}


class PagedKvCache:
    """Pools of pages ``[pages][kv_heads][page_size][head_dim]`` for keys and values in ``"f16"`` or ``"bf16"``; the
    caller's (``k_pages``, ``v_pages``: device addresses that outlive this object) or, both 0, its own, zero-filled.
    ``rope_freq``: the rotation's ``rope_dims / 2`` frequencies where they are not ``rope_base^(-2i / rope_dims)``."""

    def __init__(self, ctx: CudaContext, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: str,
                 k_pages: int = 0, v_pages: int = 0, rope_dims: int = 0, rope_interleaved: bool = False,
                 rope_base: float = 10000.0, rope_freq: Optional[Sequence[float]] = None):
        if dtype not in _DTYPES:
            raise InvalidArgument(f"dtype must be one of {sorted(_DTYPES)}, got {dtype!r}")
        freq = None if rope_freq is None else np.ascontiguousarray(rope_freq, dtype=np.float64)
        if freq is not None and freq.size != rope_dims // 2:
            raise InvalidArgument(f"rope_freq needs {rope_dims // 2} numbers, got {freq.size}")
        d = _lib.KvCacheDesc(k_pages or None, v_pages or None, pages, page_size, kv_heads, head_dim, _DTYPES[dtype], rope_dims,
                             int(rope_interleaved), rope_base, None if freq is None else _ptr(freq))
        self._h = None
        h = C.c_void_p()
        try:
            check(load().nne_kv_cache_create(ctx.handle, C.byref(d), C.byref(h)))
        except NneError as e:
            _raise_mapped(e)
        self._h, self.ctx = h, ctx
        self.pages, self.page_size, self.kv_heads, self.head_dim, self.dtype = pages, page_size, kv_heads, head_dim, dtype

    @property
    def handle(self):
        if self._h is None:
            raise GpuError("cache was closed")
        return self._h

    def pools(self):
        """(address of the keys' pool, address of the values' pool, bytes of each)."""
        k, v, n = C.c_void_p(), C.c_void_p(), C.c_size_t()
        check(load().nne_kv_cache_info(self.handle, C.byref(k), C.byref(v), C.byref(n)))
        return k.value, v.value, n.value

    def close(self):
        if getattr(self, "_h", None) is not None:
            load().nne_kv_cache_destroy(self._h)
            self._h = None

    def __del__(self):  # pragma: no cover - best effort
        try:
            self.close()
        except Exception:
            pass


class _Call:
    """An argument block over fixed device buffers and the entry point it goes to."""

    def __init__(self, entry, args):
        self._entry, self.args, self._ref = entry, args, C.byref(args)

    def _issue(self, handle, stream: int) -> None:
        status = self._entry(handle, self._ref, stream)
        if status != _lib.OK:
            _raise_mapped(NneError(status, _lib.last_error()))


class KvAppend(_Call):
    """Per-head RMSNorm and rotation of queries and keys, keys and values into their pages (``nne_kv_append_dev``).
    Strides count floats from token to token; 0 means heads without gaps."""

    def __init__(self, cache: PagedKvCache, tokens: int, q_heads: int = 0, q: int = 0, k: int = 0, v: int = 0, q_out: int = 0,
                 q_stride: int = 0, k_stride: int = 0, v_stride: int = 0, q_gamma: int = 0, k_gamma: int = 0, eps: float = 1e-6,
                 page_table: int = 0, table_stride: int = 0, sequences: int = 0, sequence: int = 0, index: int = 0,
                 position: int = 0):
        kv = cache.kv_heads * cache.head_dim
        super().__init__(load().nne_kv_append_dev, _lib.KvAppendArgs(
            q or None, k or None, v or None, q_out or None, q_stride or q_heads * cache.head_dim, k_stride or kv, v_stride or kv,
            tokens, q_heads, eps, q_gamma or None, k_gamma or None, page_table or None, table_stride, sequences, sequence or None,
            index or None, position or None))
        self.cache = cache

    def run(self, stream: int = 0) -> None:
        self._issue(self.cache.handle, stream)


class TreeAttention(_Call):
    """Attention of the newest tokens of each sequence over the cache (``nne_tree_attention_dev``): a tree of up to 64
    drafted nodes, a chain (``visible`` 0) or, one node a sequence, ordinary decoding.  ``node_start`` i32
    ``[sequences + 1]``, ``context`` i32 ``[sequences]``, ``visible`` u64 ``[tokens]``; ``scale`` defaults to
    ``head_dim ** -0.5``."""

    def __init__(self, cache: PagedKvCache, tokens: int, q_heads: int, q: int, out: int, sequences: int, node_start: int, context: int,
                 page_table: int, table_stride: int, max_nodes: int, max_context: int, visible: int = 0, scale: Optional[float] = None,
                 q_stride: int = 0, out_stride: int = 0):
        width = q_heads * cache.head_dim
        super().__init__(load().nne_tree_attention_dev, _lib.TreeAttentionArgs(
            q or None, out or None, q_stride or width, out_stride or width, tokens, q_heads, sequences, max_nodes, max_context,
            cache.head_dim ** -0.5 if scale is None else scale, node_start or None, context or None, visible or None,
            page_table or None, table_stride))
        self.cache = cache

    def run(self, stream: int = 0) -> None:
        self._issue(self.cache.handle, stream)


class Sampler(_Call):
    """One token a row of logits, from given uniform numbers (``nne_sample_dev``).  ``temperature``, ``top_k`` (i32),
    ``top_p`` and ``min_p`` are addresses of one setting a row, 0 for "off"; ``tokens`` i32 ``[rows]``."""

    def __init__(self, ctx: CudaContext, rows: int, vocab: int, logits: int, uniform: int, tokens: int, temperature: int = 0,
                 top_k: int = 0, top_p: int = 0, min_p: int = 0, row_stride: int = 0):
        super().__init__(load().nne_sample_dev, _lib.SampleArgs(
            logits or None, row_stride or vocab, rows, vocab, temperature or None, top_k or None, top_p or None, min_p or None,
            uniform or None, tokens or None))
        self.ctx = ctx

    def run(self, stream: int = 0) -> None:
        self._issue(self.ctx.handle, stream)
