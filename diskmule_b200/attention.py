"""Attention and its paged key/value cache over the C ABI (include/diskmule_attention.h).

`prompt_attention` runs whole prompts, `KvCache` holds the pages of many sequences and
`KvCache.decode_attention` runs one query token per sequence against them. Every tensor and
list is a device pointer (an int); strides are in elements. Calls are ordered on `stream`
(0: the default stream) and allocate nothing.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _native as N
from ._native import check
from .moe import CudaContext


def _strides(pair):  # zeros: contiguous
    return (C.c_int64 * 2)() if pair is None else (C.c_int64 * 2)(*pair)


def prompt_attention(ctx: CudaContext, *, type: int, heads: int, kv_heads: int, head_dim: int,
                     q: int, k: int, v: int, out: int, q_tokens: int, k_tokens: int,
                     sequences: int, q_offsets: int, k_offsets: int = 0, lse: int = 0,
                     causal: bool = True, window: int = 0, scale: float = 0.0, q_stride=None,
                     k_stride=None, v_stride=None, out_stride=None, stream: int = 0):
    """Packed attention of `sequences` prompts (dm_attention_prompt). `*_stride` are
    (token, head) pairs, None for contiguous tensors; scale 0 is 1 / sqrt(head_dim)."""
    d = N.PromptDesc(type, heads, kv_heads, head_dim, sequences, int(causal), window, scale,
                     q_tokens, k_tokens, q, k, v, out, lse or None)
    d.q_offsets = q_offsets
    d.k_offsets = k_offsets or None
    if q_stride or k_stride or v_stride or out_stride:
        d.q_stride, d.k_stride = _strides(q_stride), _strides(k_stride)
        d.v_stride, d.out_stride = _strides(v_stride), _strides(out_stride)
    check(N.lib().dm_attention_prompt(ctx.handle, C.byref(d), stream or None))


def attention_status(ctx: CudaContext, stream: int = 0):
    """Wait for `stream`; raises if a bounded wait inside an attention kernel ran out."""
    check(N.lib().dm_attention_status(ctx.handle, stream or None))


class KvCache:
    """A paged key/value cache (dm_kv_cache). `memory`, `page_table`, `lengths` and
    `references` are device pointers that the caller keeps alive, or 0 to let the cache
    allocate them."""

    def __init__(self, ctx: CudaContext, *, type: int, layers: int, kv_heads: int, head_dim: int,
                 page_tokens: int, pages: int, max_sequences: int, max_pages: int,
                 memory: int = 0, page_table: int = 0, lengths: int = 0, references: int = 0):
        self._h = None
        self._ctx = ctx
        self._lib = N.lib()
        d = N.KvCacheDesc(type, layers, kv_heads, head_dim, page_tokens, pages, max_sequences,
                          max_pages, memory or None, page_table or None, lengths or None,
                          references or None)
        h = C.c_void_p()
        check(N.lib().dm_kv_cache_create(ctx.handle, C.byref(d), C.byref(h)))
        self._h = h

    @property
    def handle(self):
        return self._h

    def describe(self) -> N.KvCacheDesc:
        d = N.KvCacheDesc()
        check(self._lib.dm_kv_cache_describe(self._h, C.byref(d)))
        return d

    def status(self, stream: int = 0) -> int:
        """Wait for `stream`; the KV_* bits since the last call."""
        bits = C.c_int32(0)
        check(self._lib.dm_kv_cache_status(self._h, C.byref(bits), stream or None))
        return bits.value

    def extend(self, sequences: int, counts: int, n: int, stream: int = 0):
        check(self._lib.dm_kv_cache_extend(self._h, sequences, counts, n, stream or None))

    def write(self, layer: int, k: int, v: int, sequences: int, offsets: int, n: int, tokens: int,
              k_stride=None, v_stride=None, stream: int = 0):
        check(self._lib.dm_kv_cache_write(
            self._h, layer, k, v, None if k_stride is None else _strides(k_stride),
            None if v_stride is None else _strides(v_stride), sequences, offsets, n, tokens,
            stream or None))

    def fork(self, parents: int, children: int, n: int, stream: int = 0):
        check(self._lib.dm_kv_cache_fork(self._h, parents, children, n, stream or None))

    def compact(self, sequences: int, keep_offsets: int, keep: int, n: int, kept: int,
                stream: int = 0):
        check(self._lib.dm_kv_cache_compact(self._h, sequences, keep_offsets, keep, n, kept,
                                          stream or None))

    def free(self, sequences: int, n: int, stream: int = 0):
        check(self._lib.dm_kv_cache_free(self._h, sequences, n, stream or None))

    def copy_pages(self, source: int, target: int, n: int, stream: int = 0):
        check(self._lib.dm_kv_cache_copy_pages(self._h, source, target, n, stream or None))

    def decode_workspace(self, heads: int, batch: int, shared_tokens: int, max_length: int) -> int:
        """Bytes of workspace that decode_attention needs for these numbers."""
        n = C.c_uint64(0)
        check(self._lib.dm_attention_decode_workspace(self._h, heads, batch, shared_tokens,
                                                    max_length, C.byref(n)))
        return n.value

    def decode_attention(self, *, layer: int, heads: int, q: int, out: int, batch: int,
                         max_length: int, shared_tokens: int = 0, sequences: int = 0, lse: int = 0,
                         window: int = 0, scale: float = 0.0, q_stride=None, out_stride=None,
                         workspace: int = 0, workspace_bytes: int = 0, stream: int = 0):
        """One query token per sequence over the cache (dm_attention_decode)."""
        d = N.DecodeDesc(layer, heads, batch, window, shared_tokens, max_length, scale, q, out,
                         lse or None)
        d.sequences = sequences or None
        d.workspace = workspace or None
        d.workspace_bytes = workspace_bytes
        if q_stride or out_stride:
            d.q_stride, d.out_stride = _strides(q_stride), _strides(out_stride)
        check(self._lib.dm_attention_decode(self._h, C.byref(d), stream or None))

    def close(self):
        if self._h:
            self._lib.dm_kv_cache_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def offsets(lengths) -> np.ndarray:
    """int32 offsets of packed sequences, [len(lengths) + 1]."""
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
