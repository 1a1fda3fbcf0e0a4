"""QuantizedKvCache: keys and values of a model's attention layers in 8 bits, and attention over them.

One object holds every layer's cache of a batch of sequences and the device array of their lengths.  A step stores its
tokens layer by layer, attends, and advances the lengths once at the end:

    cache = QuantizedKvCache(lane, layers, sequences, kv_heads, head_width, capacity)
    for layer in range(layers):
        cache.store(layer, k, v, tokens, q=q, q_out=q, heads=heads, rotary=rotary)
        cache.attention(layer, q, heads, tokens, out=context)
    cache.advance(tokens)

Lengths live on the device, so a captured graph of such a step serves every position.  It stands where the reference's
attention step keeps its key/value buffers (Qwen35Gpu.AttentionStep, NNtrain.Core/Modules/Qwen35Gpu.Attention.cs:60-120).
"""
from __future__ import annotations

import ctypes
import math
import struct
from ctypes import byref, c_uint64

import numpy as np

from .lane import HipBuffer, HipExecutionLane
from .native import (KV_BLOCK_TOKENS, ROTARY_HALVES, ROTARY_PAIRS, AttentionDesc, KvCacheDesc, KvStoreDesc, RowsDesc, check)


# The native descriptors are filled in one go: a token step makes these calls for every layer, and field by field they take
# longer on the host than the launches on the device.
_STORE, _ATTENTION, _ROWS = struct.Struct("=Ii Q Qqq Qqq Qqq Qqq Q iIiI"), struct.Struct("=Ii Q Qqq Qqq iiif"), struct.Struct("=Qqq")
assert _STORE.size == ctypes.sizeof(KvStoreDesc) and _ATTENTION.size == ctypes.sizeof(AttentionDesc)
_NO_ROWS = (0, 0, 0)
_LARGEST = 2**31 - 1


class Rows:
    """FP32 rows [sequence, token, width] inside a buffer: element (b, i, c) lies at offset + b * sequence_stride +
    i * token_stride + c, all in floats.  A plain HipBuffer stands for dense rows."""
    __slots__ = ("buffer", "token_stride", "sequence_stride", "offset")

    def __init__(self, buffer: HipBuffer, token_stride: int, sequence_stride: int = 0, offset: int = 0):
        if token_stride < 0 or sequence_stride < 0 or offset < 0:
            raise ValueError("strides and offset must not be negative.")
        self.buffer, self.token_stride, self.sequence_stride, self.offset = buffer, token_stride, sequence_stride, offset


class Rotary:
    """Rotary positions: pair j of a head's first `width` components turns by position * inv_freq[j] (inv_freq: FP32 on the
    device, width / 2 values).  pairs=False: pair j is (j, j + width / 2); pairs=True: (2j, 2j + 1)."""
    __slots__ = ("inv_freq", "width", "style")

    def __init__(self, inv_freq: HipBuffer, width: int, pairs: bool = False):
        if width < 2 or width % 2 != 0:
            raise ValueError("the rotary width must be even and positive.")
        if inv_freq.nbytes < 2 * width:
            raise ValueError("inv_freq holds fewer than width / 2 values.")
        self.inv_freq, self.width, self.style = inv_freq, width, ROTARY_PAIRS if pairs else ROTARY_HALVES

    @staticmethod
    def frequencies(width: int, base: float = 10000.0) -> np.ndarray:
        """base^(-2j / width), the usual choice."""
        return (base ** (-np.arange(0, width, 2, dtype=np.float64) / width)).astype(np.float32)


class QuantizedKvCache:
    BLOCK_TOKENS = KV_BLOCK_TOKENS

    def __init__(self, lane: HipExecutionLane, layers: int, sequences: int, kv_heads: int, head_width: int, capacity: int):
        if min(layers, sequences, kv_heads, head_width, capacity) <= 0:
            raise ValueError("layers, sequences, kv_heads, head_width and capacity must be positive.")
        size = c_uint64()
        check(lane._lib.nnhip_kv_cache_bytes(sequences, kv_heads, head_width, capacity, byref(size)), "kv_cache_bytes")
        self.lane, self.layers, self.sequences = lane, layers, sequences
        self.kv_heads, self.head_width, self.capacity = kv_heads, head_width, capacity
        self.layer_bytes = size.value
        self._owned: list[HipBuffer] = []
        try:
            self.lengths = lane.allocate_bytes(4 * sequences)
            self._owned.append(self.lengths)
            for _ in range(layers):
                self._owned.append(lane.allocate_bytes(self.layer_bytes))
        except BaseException:
            self.dispose()
            raise
        self._caches = [KvCacheDesc(ctypes.sizeof(KvCacheDesc), sequences, kv_heads, head_width, capacity, 0, b.ptr, self.lengths.ptr)
                        for b in self._owned[1:]]
        self._refs = [byref(c) for c in self._caches]
        self._store, self._attention, self._k_out, self._v_out = KvStoreDesc(), AttentionDesc(), RowsDesc(), RowsDesc()
        self.reset()

    # ---- lengths ----
    def reset(self) -> None:
        """Every sequence empty."""
        self._cache(0)
        self.lane.fill_u32(self.lengths, 0, self.sequences)

    def set_lengths(self, lengths) -> None:
        """The tokens each sequence holds; smaller than before drops the last ones."""
        self._cache(0)
        values = np.asarray(lengths)            # (checked before they are made 32 bits wide)
        if values.dtype.kind not in "biuf" or values.shape != (self.sequences,) or not np.all((values >= 0) & (values <= self.capacity) & (values % 1 == 0)):
            raise ValueError("lengths must be one whole number of 0 .. capacity for each sequence.")
        self.lane.write(self.lengths, values.astype(np.int32))

    def read_lengths(self) -> np.ndarray:
        self._cache(0)
        return self.lane.read(self.lengths, np.int32, self.sequences)

    def advance(self, tokens: int = 1, counts: HipBuffer | None = None) -> None:
        """Adds a step's tokens to the lengths, after its last layer."""
        cache = self._cache(0)
        with self.lane.kernel("kv_cache_advance"):
            check(self.lane._lib.nnhip_kv_cache_advance(self.lane._handle, cache, tokens, self._int32(counts, "counts") or None),
                  "kv_cache_advance")

    # ---- tokens ----
    def store(self, layer: int, k: "HipBuffer | Rows", v: "HipBuffer | Rows", tokens: int = 1, *, counts: HipBuffer | None = None,
              rotary: Rotary | None = None, q: "HipBuffer | Rows | None" = None, q_out: "HipBuffer | Rows | None" = None,
              heads: int = 0) -> None:
        """Stores `tokens` new tokens of every sequence behind its length (the first counts[b] of them with counts, int32 on
        the device), keys turned by their positions with `rotary`.  q (heads query heads of the same tokens) is turned into
        q_out, q itself by default.  A sequence whose tokens would pass the capacity is left out."""
        cache = self._cache(layer)
        if not 1 <= tokens <= _LARGEST:
            raise ValueError("tokens must be positive and fit 32 bits.")
        kv_width = self.kv_heads * self.head_width
        counts_ptr = self._int32(counts, "counts")
        k_rows, v_rows = self._rows(k, tokens, kv_width, "k"), self._rows(v, tokens, kv_width, "v")
        turn = (0, 0, 0)
        if rotary is not None:
            if rotary.width > self.head_width:
                raise ValueError("the rotary width exceeds head_width.")
            turn = rotary.inv_freq._require(), rotary.width, rotary.style
        q_rows = out_rows = _NO_ROWS
        if q is not None:
            if rotary is None or not 1 <= heads <= _LARGEST:
                raise ValueError("q needs rotary and a positive number of heads.")
            q_rows = self._rows(q, tokens, heads * self.head_width, "q")
            out_rows = q_rows if q_out is None else self._rows(q_out, tokens, heads * self.head_width, "q_out")
        elif q_out is not None or heads:
            raise ValueError("q_out and heads need q.")
        lane = self.lane
        _STORE.pack_into(self._store, 0, _STORE.size, tokens, counts_ptr, *k_rows, *v_rows, *q_rows, *out_rows, *turn, heads, 0)
        with lane.kernel("kv_cache_store"):
            check(lane._lib.nnhip_kv_cache_store(lane._handle, cache, self._store), "kv_cache_store")

    def attention(self, layer: int, q: "HipBuffer | Rows", heads: int, tokens: int = 1, *, scale: float | None = None,
                  window: int = 0, sinks: int = 0, counts: HipBuffer | None = None,
                  out: "HipBuffer | Rows | None" = None) -> "HipBuffer | Rows":
        """Causal attention of the tokens just stored over the cache: token i of sequence b stands at position lengths[b] + i
        and sees the keys up to it, with window > 0 the last `window` of them and the first `sinks` tokens.  scale: 1 /
        sqrt(head_width) by default.  FP32 in and out; rows behind counts[b] are left as they are.  The scale of a block covers
        all its stored tokens: of tokens stored together, those behind a row have that influence on it."""
        cache = self._cache(layer)
        if not 1 <= tokens <= _LARGEST or not 1 <= heads <= _LARGEST or heads % self.kv_heads != 0:
            raise ValueError("tokens must be positive, heads a positive multiple of kv_heads, both fit 32 bits.")
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks must not be negative.")
        factor = 1.0 / math.sqrt(self.head_width) if scale is None else scale
        if not 0.0 <= factor <= 1e30:
            raise ValueError("scale must be 0 .. 1e30.")
        width = heads * self.head_width
        lane, q_rows, counts_ptr = self.lane, self._rows(q, tokens, width, "q"), self._int32(counts, "counts")
        target = out if out is not None else lane.allocate(self.sequences * tokens * width)
        try:
            _ATTENTION.pack_into(self._attention, 0, _ATTENTION.size, tokens, counts_ptr, *q_rows, *self._rows(target, tokens, width, "out"),
                                 heads, min(window, _LARGEST), min(sinks, _LARGEST), factor)
            with lane.kernel("cached_attention"):
                check(lane._lib.nnhip_cached_attention(lane._handle, cache, self._attention), "cached_attention")
        except BaseException:
            if out is None:
                target.dispose()
            raise
        return target

    def read(self, layer: int, tokens: int, *, first: HipBuffer | None = None, k_out: "HipBuffer | Rows | None" = None,
             v_out: "HipBuffer | Rows | None" = None) -> None:
        """FP32 values of tokens first[b] .. first[b] + tokens - 1 of every sequence (first: int32 on the device, 0 without)."""
        cache = self._cache(layer)
        if not 1 <= tokens <= _LARGEST:
            raise ValueError("tokens must be positive and fit 32 bits.")
        if k_out is None and v_out is None:
            raise ValueError("read needs k_out or v_out.")
        width = self.kv_heads * self.head_width
        lane, first_ptr = self.lane, self._int32(first, "first")
        _ROWS.pack_into(self._k_out, 0, *(self._rows(k_out, tokens, width, "k_out") if k_out is not None else _NO_ROWS))
        _ROWS.pack_into(self._v_out, 0, *(self._rows(v_out, tokens, width, "v_out") if v_out is not None else _NO_ROWS))
        with lane.kernel("kv_cache_read"):
            check(lane._lib.nnhip_kv_cache_read(lane._handle, cache, first_ptr or None, tokens, self._k_out, self._v_out), "kv_cache_read")

    # ---- checks ----
    def _cache(self, layer: int):
        """The native descriptor of a layer's cache, by reference."""
        if not self._owned:
            raise ValueError("the cache has been disposed")
        if not 0 <= layer < self.layers:
            raise IndexError(f"layer {layer} is outside 0 .. {self.layers - 1}.")
        return self._refs[layer]

    def _int32(self, buffer: HipBuffer | None, name: str) -> int:
        if buffer is None:
            return 0
        if buffer.nbytes < 4 * self.sequences:
            raise ValueError(f"The buffer '{name}' holds fewer values than there are sequences.")
        return buffer._require()

    def _rows(self, rows: "HipBuffer | Rows", tokens: int, width: int, name: str) -> tuple[int, int, int]:
        """Pointer, token stride and sequence stride of an operand."""
        if rows is None:
            raise TypeError(f"{name} is null.")
        if isinstance(rows, Rows):
            buffer, token, sequence, offset = rows.buffer, rows.token_stride, rows.sequence_stride, rows.offset
        else:
            buffer, token, sequence, offset = rows, width, tokens * width, 0
        if buffer.nbytes < 4 * (offset + (self.sequences - 1) * sequence + (tokens - 1) * token + width):
            raise ValueError(f"The buffer '{name}' is too small for its rows.")
        return buffer._require() + 4 * offset, token, sequence

    def dispose(self) -> None:
        for b in reversed(self._owned):
            b.dispose()
        self._owned = []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.dispose()


__all__ = ["QuantizedKvCache", "Rotary", "Rows"]
