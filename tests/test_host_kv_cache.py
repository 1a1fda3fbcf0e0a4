"""CPU-side checks of the 8-bit key/value cache: sizes, the operand classes, and the block layout."""
import ctypes
from ctypes import byref, c_uint64

import numpy as np
import pytest

from nntrain_amd import HipBuffer, Rotary, Rows, native


def _bytes(*args):
    size = c_uint64()
    return native.load_library().nnhip_kv_cache_bytes(*args, byref(size)), size.value


@pytest.mark.parametrize("width,padded", [(1, 32), (32, 32), (33, 64), (80, 96), (96, 96), (128, 128), (130, 192), (200, 256), (256, 256)])
def test_cache_bytes(width, padded):
    sequences, heads, capacity = 3, 5, 130
    pairs, blocks = sequences * heads, 3
    want = 2 * pairs * blocks * 64 * padded + -(-pairs * blocks * 8 // 256) * 256 + pairs * 4 * 64 * padded * 4 + pairs * 32
    assert _bytes(sequences, heads, width, capacity) == (0, want)


def test_cache_bytes_refusals_and_sizes_behind_32_bits():
    for bad in ((0, 1, 64, 1), (1, 0, 64, 1), (1, 1, 0, 1), (1, 1, 64, 0), (-1, 1, 64, 1)):
        assert _bytes(*bad)[0] == 1, bad
    assert _bytes(1, 1, 257, 1)[0] == 8 and _bytes(2**31 - 1, 2, 64, 1)[0] == 8 and _bytes(2**20, 2**11 - 1, 256, 2**31 - 1)[0] == 8
    status, size = _bytes(32, 16, 128, 1 << 20)
    assert status == 0 and size > 2 * 32 * 16 * 128 * (1 << 20)
    assert native.load_library().nnhip_kv_cache_bytes(1, 1, 64, 1, None) == 1


def test_structure_sizes():
    assert ctypes.sizeof(native.RowsDesc) == 24 and ctypes.sizeof(native.KvCacheDesc) == 40
    assert ctypes.sizeof(native.KvStoreDesc) == 136 and ctypes.sizeof(native.AttentionDesc) == 80
    assert ctypes.sizeof(native.LogProbsDesc) == 72


def test_operand_checks():
    class NoLane:
        disposed = False
    b = HipBuffer(NoLane(), 4096, 4 * 32)
    assert Rows(b, 0, 0, 3).offset == 3 and Rotary(b, 64, pairs=True).style == native.ROTARY_PAIRS
    for bad in (lambda: Rows(b, -1), lambda: Rows(b, 1, -1), lambda: Rows(b, 1, 1, -1), lambda: Rotary(b, 0), lambda: Rotary(b, 3),
                lambda: Rotary(b, 66)):
        with pytest.raises(ValueError):
            bad()
    f = Rotary.frequencies(8, 16.0)
    assert f.dtype == np.float32 and np.allclose(f, [1.0, 0.5, 0.25, 0.125])


def test_positions_stay_away_from_the_largest_integer():
    assert _bytes(1, 1, 64, 2**30)[0] == 0 and _bytes(1, 1, 64, 2**30 + 1)[0] == 8


def test_lengths_are_checked_before_they_are_narrowed():
    from nntrain_amd import QuantizedKvCache

    class Lane:
        disposed = False

        def write(self, buffer, values):
            self.written = values
    cache = QuantizedKvCache.__new__(QuantizedKvCache)
    cache.lane, cache.layers, cache.sequences, cache.capacity, cache.lengths = Lane(), 1, 2, 100, None
    cache._owned, cache._refs = [None], [None]
    for bad in ([0, 2**32], np.array([2**32 + 5, 1]), np.array([2**64 - 1, 0], np.uint64), [1.5, 2.0], [np.nan, 0.0], [0, -1], [0, 101], [[0, 1]], [1], ["0", "1"]):
        with pytest.raises(ValueError):
            cache.set_lengths(bad)
    for good in ([0, 100], (3, 4), np.array([7, 100], np.int64), np.array([1, 2], np.uint8), np.zeros(2)):
        cache.set_lengths(good)
        assert cache.lane.written.dtype == np.int32 and list(cache.lane.written) == list(good)
