"""Attention and its paged key/value cache over the C ABI (include/diskmule_attention.h).

`prompt_attention` runs whole prompts, `KvCache` holds the pages of many sequences and
`KvCache.decode_attention` runs one query token per sequence against them,
`KvCache.chunk_attention` any number of new tokens. `rotate` norms and rotates queries and keys
on their way there, `KvCache.token_weights` sums the attention that tokens receive and
`KvCache.evict` keeps those that received most. Every tensor and list is a device pointer (an
int); strides are in elements. Calls are ordered on `stream` (0: the default stream) and
allocate nothing.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _native as N
from ._native import check
from .moe import CudaContext


_Pair = C.c_int64 * 2


def _strides(pair):  # zeros: contiguous
    return _Pair() if pair is None else _Pair(*pair)


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


class Rope:
    """Which values of a head turn with the position, and how fast (dm_rope). `frequencies`
    (radians per position, one per pair) default to theta^(-2 i / rotary_dim); `pair_axes`
    names the axis of positions that each pair turns with (all 0)."""

    def __init__(self, ctx: CudaContext, rotary_dim: int, *, theta: float = 10000.0, frequencies=None,
                 pair_axes=None, axes: int = 0, interleaved: bool = False, scale: float = 1.0):
        self._h = None
        self._ctx = ctx
        self._lib = N.lib()
        half = rotary_dim // 2
        f = a = None
        if frequencies is not None:
            f = np.ascontiguousarray(frequencies, np.float64)
        if pair_axes is not None:
            a = np.ascontiguousarray(pair_axes, np.int32)
        for given in (f, a):
            if given is not None and given.shape != (half,):
                raise ValueError(f"{half} pairs, and values of shape {given.shape}")
        self.axes = axes or (1 if a is None else int(a.max(initial=0)) + 1)
        d = N.RopeDesc(rotary_dim, int(interleaved), self.axes, scale, theta)
        if f is not None:
            d.frequencies = f.ctypes.data_as(C.POINTER(C.c_double))
        if a is not None:
            d.pair_axes = a.ctypes.data_as(C.POINTER(C.c_int32))
        h = C.c_void_p()
        check(self._lib.dm_rope_create(ctx.handle, C.byref(d), C.byref(h)))
        self._h = h

    @property
    def handle(self):
        return self._h

    def close(self):
        if self._h:
            self._lib.dm_rope_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def rotate(ctx: CudaContext, rope: Rope | None, *, type: int, head_dim: int, tokens: int, heads: int = 0,
           kv_heads: int = 0, q: int = 0, k: int = 0, v: int = 0, q_out: int = 0, k_out: int = 0,
           v_out: int = 0, cache: KvCache | None = None, layer: int = 0, sequences: int = 0,
           offsets: int = 0, n: int = 0, positions: int = 0, norm_q: bool = False, norm_k: bool = False,
           norm_v: bool = False, q_weight: int = 0, k_weight: int = 0, epsilon: float = 1e-6,
           q_stride=None, k_stride=None, v_stride=None, q_out_stride=None, k_out_stride=None,
           v_out_stride=None, stream: int = 0):
    """Norm each head and rotate queries and keys, into `*_out` and, with a cache, keys and values
    into its pages as the last tokens of `sequences` (dm_attention_rotate)."""
    # null would mean that none is wanted
    if rope is not None and not rope._h or cache is not None and not cache._h:
        raise N.DmError(N.ERR_INVALID_ARGUMENT, "a closed rotation or cache")
    norms = norm_q * N.NORM_Q | norm_k * N.NORM_K | norm_v * N.NORM_V
    d = N.RotateDesc(type, heads, kv_heads, head_dim, norms, epsilon, layer, n, tokens, q or None, k or None,
                     v or None, q_out or None, k_out or None, v_out or None)
    if q_stride:
        d.q_stride = _Pair(*q_stride)
    if k_stride:
        d.k_stride = _Pair(*k_stride)
    if v_stride:
        d.v_stride = _Pair(*v_stride)
    if q_out_stride:
        d.q_out_stride = _Pair(*q_out_stride)
    if k_out_stride:
        d.k_out_stride = _Pair(*k_out_stride)
    if v_out_stride:
        d.v_out_stride = _Pair(*v_out_stride)
    if q_weight:
        d.q_weight = q_weight
    if k_weight:
        d.k_weight = k_weight
    if positions:
        d.positions = positions
    if sequences:
        d.rows = sequences
    if offsets:
        d.offsets = offsets
    check(N.lib().dm_attention_rotate(ctx.handle, rope._h if rope else None, cache._h if cache else None, C.byref(d),
                                      stream or None))


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

    def chunk_workspace(self, heads: int, n: int, tokens: int, max_length: int, window: int = 0,
                        sinks: int = 0) -> int:
        """Bytes of workspace that chunk_attention needs for these numbers."""
        d = N.ChunkDesc(0, heads, n, window, sinks, max_length, 0.0, tokens)
        size = C.c_uint64(0)
        check(self._lib.dm_attention_chunk_workspace(self._h, C.byref(d), C.byref(size)))
        return size.value

    def chunk_attention(self, *, layer: int, heads: int, q: int, out: int, offsets: int, n: int,
                        tokens: int, max_length: int, sequences: int = 0, lse: int = 0, window: int = 0,
                        sinks: int = 0, scale: float = 0.0, q_stride=None, out_stride=None,
                        workspace: int = 0, workspace_bytes: int = 0, stream: int = 0):
        """The last offsets[i + 1] - offsets[i] tokens of each of `n` sequences over the cache
        (dm_attention_chunk)."""
        d = N.ChunkDesc(layer, heads, n, window, sinks, max_length, scale, tokens, q, out, lse or None)
        d.rows, d.offsets = sequences or None, offsets
        d.workspace, d.workspace_bytes = workspace or None, workspace_bytes
        if q_stride or out_stride:
            d.q_stride, d.out_stride = _strides(q_stride), _strides(out_stride)
        check(self._lib.dm_attention_chunk(self._h, C.byref(d), stream or None))

    def token_weights(self, *, layer: int, heads: int, q: int, lse: int, offsets: int, n: int, tokens: int,
                      max_length: int, weights: int, weights_stride: int, sequences: int = 0, window: int = 0,
                      sinks: int = 0, scale: float = 0.0, q_stride=None, stream: int = 0):
        """Add the attention that cached tokens get from these queries to `weights`, f32
        [max_sequences, weights_stride] (dm_attention_weights)."""
        d = N.WeightsDesc(layer, heads, n, window, sinks, max_length, scale, tokens, q, lse)
        if q_stride:
            d.q_stride = _strides(q_stride)
        d.rows, d.offsets = sequences or None, offsets
        d.weights, d.weights_stride = weights, weights_stride
        check(self._lib.dm_attention_weights(self._h, C.byref(d), stream or None))

    def evict(self, *, sequences: int, n: int, budget: int, weights: int, weights_stride: int,
              keep_offsets: int, keep: int, sinks: int = 0, recent: int = 0, stream: int = 0):
        """Keep `budget` tokens of each sequence: the first `sinks`, the last `recent` and the
        heaviest between (dm_kv_cache_evict)."""
        d = N.EvictDesc(n, budget, sinks, recent, sequences, weights, weights_stride, keep_offsets, keep)
        check(self._lib.dm_kv_cache_evict(self._h, C.byref(d), stream or None))

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
