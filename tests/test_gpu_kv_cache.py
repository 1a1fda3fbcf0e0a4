"""The 8-bit key/value cache and attention over it, through the package, against the 64-bit restatement.

Bars.  Stored values: without rotary positions the codes and scales are a function of the FP32 inputs, so values are equal bit
for bit.  With them, a key component is a 64-bit value rounded once; two implementations of sine and cosine may round it to
neighbouring FP32 numbers (about one component in 2^28), and one of those may fall on the other side of a rounding border
of the codes: at most one value in 10^5 may be one step off, none more.

Attention, for n visible keys of head width w, A = the largest scale * sum |q_d K_d| of the call, M = the largest |V|:
a score is off by at most A * (2 * 2^-22 (two half-precision parts of q) + w * 2^-24 (accumulation) + 4 * 2^-24 (factors)), an
exponential of it by that plus 4 * 2^-24, numerator and denominator by n * 2^-24 more for their sums and 2^-21 for the two
parts of a probability; the quotient by the sum of both, and 2^-24 M.
"""
import numpy as np
import pytest

import kv_reference as ref
from nntrain_amd import HipExecutionLane, NnHipError, QuantizedKvCache, Rotary, Rows
from nntrain_amd.native import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lane():
    with HipExecutionLane(0) as ln:
        yield ln


def _rng(*seed):
    return np.random.default_rng(list(seed))


def _values(rng, tokens, heads, width):
    x = rng.standard_normal((tokens, heads, width)) * np.exp(0.7 * rng.standard_normal((heads, width)))
    return x.astype(np.float32)


def _read(lane, cache, layer, tokens, first=None):
    shape = (cache.sequences, tokens, cache.kv_heads, cache.head_width)
    k, v = lane.allocate(int(np.prod(shape))), lane.allocate(int(np.prod(shape)))
    f = lane.upload_raw(np.asarray(first, np.int32)) if first is not None else None
    cache.read(layer, tokens, first=f, k_out=k, v_out=v)
    out = lane.read(k).reshape(shape), lane.read(v).reshape(shape)
    for b in (k, v, f):
        if b is not None:
            b.dispose()
    return out


def _put(lane, cache, layer, k, v, **kw):
    """k, v [sequences, tokens, heads, width] stored at the present lengths."""
    kb, vb = lane.upload_raw(k), lane.upload_raw(v)
    cache.store(layer, kb, vb, k.shape[1], **kw)
    lane.synchronize()
    kb.dispose()
    vb.dispose()


def _tolerance(reach, keys, width, largest):
    score = reach * (2 * 2.0 ** -22 + width * 2.0 ** -24 + 4 * 2.0 ** -24) + 4 * 2.0 ** -24
    return (2 * (score + keys * 2.0 ** -24) + 2.0 ** -21 + 2.0 ** -24) * largest


# --------------------------------------------------------------------------------------------------------------- store
@pytest.mark.parametrize("width", [1, 20, 32, 64, 80, 96, 128, 130, 192, 256])
def test_stored_values_are_the_block_quantisation_bit_for_bit(lane, width):
    B, kv, n = 2, 3, 131
    rng = _rng(1, width)
    k, v = _values(rng, B * n, kv, width).reshape(B, n, kv, width), _values(rng, B * n, kv, width).reshape(B, n, kv, width)
    v[0, 64:128, 1] = 0.0                                           # a block of zeros
    with QuantizedKvCache(lane, 2, B, kv, width, 200) as cache:
        _put(lane, cache, 1, k, v)
        got_k, got_v = _read(lane, cache, 1, n)
        for b in range(B):
            assert np.array_equal(got_k[b], ref.cached(k[b])) and np.array_equal(got_v[b], ref.cached(v[b]))


@pytest.mark.parametrize("pieces", [[1] * 70, [63, 1, 1], [64, 64], [40, 100, 3], [1, 128, 1], [65, 62, 2], [129], [66], [3, 190]])
def test_the_cache_does_not_depend_on_how_the_tokens_arrive(lane, pieces):
    B, kv, width, n = 1, 2, 64, sum(pieces)
    rng = _rng(2, n)
    k, v = _values(rng, n, kv, width)[None], _values(rng, n, kv, width)[None]
    k *= np.linspace(0.2, 3.0, n, dtype=np.float32)[None, :, None, None]        # magnitudes grow inside a block
    inv = Rotary.frequencies(width)
    freq = lane.upload_raw(inv)
    with QuantizedKvCache(lane, 1, B, kv, width, n) as cache:
        at = 0
        for p in pieces:
            _put(lane, cache, 0, k[:, at:at + p], v[:, at:at + p])
            cache.advance(p)
            at += p
            got_k, got_v = _read(lane, cache, 0, at)
            assert np.array_equal(got_k[0], ref.cached(k[0, :at])), (p, at)
            assert np.array_equal(got_v[0], ref.cached(v[0, :at])), (p, at)
        assert list(cache.read_lengths()) == [n]
        # with rotary positions: the same cache as in one piece, bit for bit
        cache.reset()
        _put(lane, cache, 0, k, v, rotary=Rotary(freq, width))
        whole = _read(lane, cache, 0, n)
        cache.reset()
        at = 0
        for p in pieces:
            _put(lane, cache, 0, k[:, at:at + p], v[:, at:at + p], rotary=Rotary(freq, width))
            cache.advance(p)
            at += p
        for a, b in zip(whole, _read(lane, cache, 0, n)):
            assert np.array_equal(a, b)
    freq.dispose()


@pytest.mark.parametrize("width,rotary,pairs,start", [(64, 64, False, 0), (128, 128, False, 100000), (128, 64, True, 1000003), (80, 20, False, 77),
                                                      (96, 96, True, 5), (33, 2, False, 63), (256, 256, False, 8191)])
def test_rotary_positions_of_queries_and_keys(lane, width, rotary, pairs, start):
    kv, heads, n = 2, 6, 70
    rng = _rng(3, width, start)
    k, v, q = _values(rng, n, kv, width), _values(rng, n, kv, width), _values(rng, n, heads, width)
    inv = Rotary.frequencies(rotary, 500000.0)
    pos = np.arange(start, start + n)
    first = start // 64 * 64
    with QuantizedKvCache(lane, 1, 1, kv, width, start + n) as cache:
        # tokens of the open block in front of `start` go in first, so that its scale is known
        lead = _values(rng, start - first, kv, width) if start > first else None
        freq, qb = lane.upload_raw(inv), lane.upload_raw(q)
        rot = Rotary(freq, rotary, pairs)
        if lead is not None:
            cache.set_lengths([first])
            _put(lane, cache, 0, lead[None], lead[None], rotary=rot)
        cache.set_lengths([start])
        _put(lane, cache, 0, k[None], v[None], rotary=rot, q=qb, heads=heads)
        got_q = lane.read(qb).reshape(q.shape)
        want_q = ref.rotate(q, pos, inv, rotary, pairs)
        assert np.abs(got_q - want_q).max() <= 2.0 ** -23 * np.abs(q).max() * 2
        assert np.mean(got_q != want_q) < 1e-5
        assert np.array_equal(got_q[..., rotary:], q[..., rotary:])
        turned, plain = ref.rotate(k, pos, inv, rotary, pairs), v
        if lead is not None:
            turned = np.concatenate([ref.rotate(lead, np.arange(first, start), inv, rotary, pairs), turned])
            plain = np.concatenate([lead, v])
        got_k, got_v = _read(lane, cache, 0, start + n - first, first=[first])
        want_k = ref.cached(turned)
        step = np.abs(turned).max() / 127
        assert np.abs(got_k[0] - want_k).max() <= step * (1 + 2.0 ** -20) and np.mean(got_k[0] != want_k) < 1e-5
        assert np.array_equal(got_v[0], ref.cached(plain))
        for b in (freq, qb):
            b.dispose()


def test_counts_strides_and_left_out_sequences(lane):
    B, kv, heads, width, n, capacity = 6, 2, 4, 64, 9, 100
    row = (heads + 2 * kv) * width                                  # a stacked q | k | v projection, token after token
    rng = _rng(4)
    qkv = rng.standard_normal((n, B, row)).astype(np.float32)       # tokens outside, sequences inside
    counts, start = np.array([9, 0, 4, 9, -3, 50], np.int32), np.array([3, 5, 62, 95, 7, 60], np.int32)   # 3: past the capacity
    inv = Rotary.frequencies(width)
    with QuantizedKvCache(lane, 1, B, kv, width, capacity) as cache:
        zero = np.zeros((B, capacity, kv, width), np.float32)
        _put(lane, cache, 0, zero, zero)
        cache.set_lengths(start)
        buf, cb, freq = lane.upload_raw(qkv), lane.upload_raw(counts), lane.upload_raw(inv)
        part = lambda at: Rows(buf, B * row, row, at)               # noqa: E731
        cache.store(0, part(heads * width), part((heads + kv) * width), n, counts=cb, rotary=Rotary(freq, width), q=part(0), heads=heads)
        out = lane.upload_raw(np.full((B, n, heads, width), 7.0, np.float32))
        cache.attention(0, part(0), heads, n, counts=cb, out=out)
        got_k, got_v = _read(lane, cache, 0, capacity)
        now = lane.read(buf).reshape(n, B, row)
        ctx = lane.read(out).reshape(B, n, heads, width)
        for b in range(B):
            c = int(np.clip(counts[b], 0, n))
            c = c if start[b] + c <= capacity else 0
            if b == 3:
                assert np.isnan(ctx[b]).all()
            else:
                assert np.isfinite(ctx[b]).all() and np.all(ctx[b, c:] == 7.0)
            assert np.array_equal(now[c:, b], qkv[c:, b])           # rows behind the sequence's tokens stay
            want = ref.rotate(qkv[:c, b, :heads * width].reshape(c, heads, width), np.arange(start[b], start[b] + c), inv, width)
            assert np.allclose(now[:c, b, :heads * width].reshape(c, heads, width), want, rtol=2e-7, atol=1e-6)
            assert np.array_equal(now[:, b, heads * width:], qkv[:, b, heads * width:])
            stored = np.zeros((start[b] + c, kv, width), np.float32)
            stored[start[b]:] = qkv[:c, b, (heads + kv) * width:].reshape(c, kv, width)
            assert np.array_equal(got_v[b, :start[b] + c], ref.cached(stored))
            if c == 0:
                assert not got_v[b].any() and not got_k[b].any()
        cache.advance(n, cb)
        assert list(cache.read_lengths()) == [12, 5, 66, 95, 7, 69]
        for x in (buf, cb, freq, out):
            x.dispose()


def test_values_that_are_not_finite_and_tiny_and_large_ones(lane):
    kv, width, n = 2, 64, 130
    rng = _rng(5)
    k, v = _values(rng, n, kv, width), _values(rng, n, kv, width)
    k[3, 0, 5], v[70, 1, 0], v[129, 0, 1] = np.nan, np.inf, -np.inf
    k[64:128, 1] *= np.float32(1e-42)                               # subnormal magnitudes
    v[0:64, 0] *= np.float32(1e36)
    with QuantizedKvCache(lane, 1, 1, kv, width, n) as cache:
        _put(lane, cache, 0, k[None], v[None])
        got_k, got_v = _read(lane, cache, 0, n)
        assert np.array_equal(got_k[0], ref.cached(k), equal_nan=True) and np.array_equal(got_v[0], ref.cached(v), equal_nan=True)
        # token by token: the block's scale is NaN from the token on that is not finite
        cache.reset()
        for t in range(5):
            _put(lane, cache, 0, k[None, t:t + 1], v[None, t:t + 1])
            cache.advance(1)
        got_k, got_v = _read(lane, cache, 0, 5)
        assert np.array_equal(got_k[0], ref.cached(k[:5]), equal_nan=True) and np.array_equal(got_v[0], ref.cached(v[:5]))


def test_lengths_set_back_inside_and_before_the_open_block(lane):
    kv, width = 2, 64
    rng = _rng(6)
    a, b, c = (_values(rng, 150, kv, width) for _ in range(3))
    a[140:] *= 50                                                   # the tokens dropped below carry the largest values
    with QuantizedKvCache(lane, 1, 1, kv, width, 200) as cache:
        _put(lane, cache, 0, a[None], a[None])
        cache.set_lengths([135])                                    # inside the open block: as if the rest had never come
        _put(lane, cache, 0, b[None, :2], b[None, :2])
        cache.advance(2)
        got, _ = _read(lane, cache, 0, 137)
        assert np.array_equal(got[0], ref.cached(np.concatenate([a[:135], b[:2]])))
        cache.set_lengths([70])                                     # in a full block: its tokens count with their 8-bit values
        _put(lane, cache, 0, c[None, :1], c[None, :1])
        got, _ = _read(lane, cache, 0, 71)
        kept = np.concatenate([a[:64], ref.cached(a[:128])[64:70], c[:1]])
        assert np.array_equal(got[0], ref.cached(kept))
        cache.set_lengths([0])
        _put(lane, cache, 0, b[None, :65], c[None, :65])
        got_k, got_v = _read(lane, cache, 0, 65)
        assert np.array_equal(got_k[0], ref.cached(b[:65])) and np.array_equal(got_v[0], ref.cached(c[:65]))


def test_tokens_written_over_after_lengths_were_set_back_do_not_come_back(lane):
    """A call that fills up a block and goes on leaves that block's FP32 values behind; only those before it still count."""
    kv, width = 2, 64
    rng = _rng(60)
    a, b, c = (_values(rng, 200, kv, width) for _ in range(3))
    a[32:64] *= 100
    with QuantizedKvCache(lane, 1, 1, kv, width, 256) as cache:
        def put(at, x):
            cache.set_lengths([at])
            _put(lane, cache, 0, x[None], x[None])
            return _read(lane, cache, 0, at + len(x))[0][0]

        put(0, a[:32])
        put(32, a[32:96])                                           # into the next block
        got = put(32, b[:1])                                        # the dropped tokens' scale goes with them
        assert np.array_equal(got, ref.cached(np.concatenate([a[:32], b[:1]])))
        put(10, b[:100])                                            # over the first block, whose values a buffer holds
        full = np.concatenate([a[:10], b[:54]])
        got = put(25, c[:1])
        assert np.array_equal(got, ref.cached(np.concatenate([ref.cached(full)[:25], c[:1]])))
        # a block in the middle of a call, held by a buffer from before
        cache.reset()
        put(0, a[:100])
        put(100, a[100:190])                                        # the buffers hold blocks 1 and 2
        put(3, b[:187])
        for at in (150, 80):
            whole = ref.cached(np.concatenate([a[:3], b[:187]])[at // 64 * 64:at // 64 * 64 + 64])
            got = put(at, c[:1])
            if at < 128:
                assert np.array_equal(got[64:], ref.cached(np.concatenate([whole[:at - 64], c[:1]])))
            else:
                kept = np.concatenate([a[:3], b[:187]])[128:at]
                assert np.array_equal(got[128:], ref.cached(np.concatenate([kept, c[:1]])))


@pytest.mark.parametrize("seed", range(6))
def test_lengths_set_back_again_and_again(lane, seed):
    """Every token stays within what its quantisations can move it: half a step of its block each, at most one a store that
    reached the block (and FP32 roundings, 2^-22 of the largest)."""
    kv, width, capacity = 1, 32, 400
    rng = _rng(61, seed)
    truth = np.zeros((capacity, kv, width), np.float32)
    touched, largest = np.zeros(7, int), np.zeros(7)
    with QuantizedKvCache(lane, 1, 1, kv, width, capacity) as cache:
        length = 0
        for _ in range(40):
            if rng.random() < 0.5:
                length = max(0, length - int(rng.integers(1, 150)))
            n = min(int(rng.choice([1, 1, 3, 8, 9, 40, 64, 100, 150])), capacity - length)
            if n == 0:
                continue
            x = _values(rng, n, kv, width)
            cache.set_lengths([length])
            _put(lane, cache, 0, x[None], x[None])
            truth[length:length + n] = x
            for block in range(length // 64, (length + n - 1) // 64 + 1):
                fresh = length <= block * 64
                now = np.abs(x[max(0, block * 64 - length):block * 64 + 64 - length]).max()
                touched[block], largest[block] = (1, now) if fresh else (touched[block] + 1, max(largest[block], now))
            length += n
            for got in _read(lane, cache, 0, length):
                for block in range((length + 63) // 64):
                    off = np.abs(got[0] - truth[:length])[block * 64:block * 64 + 64].max()
                    steps = 0.5 / 127 * (1 + 1 / 127) ** touched[block]         # (a quantised value may exceed its own by half a step)
                    assert off <= touched[block] * largest[block] * (steps + 2.0 ** -22), (seed, length, block)


def test_read_outside_the_capacity_and_behind_the_last_token(lane):
    with QuantizedKvCache(lane, 1, 2, 1, 64, 70) as cache:
        x = _values(_rng(7), 10, 1, 64)
        _put(lane, cache, 0, np.stack([x, x]), np.stack([x, x]))
        k, v = _read(lane, cache, 0, 12, first=[-2, 4])
        assert not k[0, :2].any() and np.array_equal(k[0, 2:], ref.cached(x)) and np.array_equal(v[1, :6], ref.cached(x)[4:])
        assert not v[1, 6:].any()                                   # the rest of the last block
        k, _ = _read(lane, cache, 0, 20, first=[65, 2**31 - 5])
        assert not k[0, 5:].any() and not k[1].any()


# --------------------------------------------------------------------------------------------------------------- attention
CASES = [  # heads, kv_heads, width, tokens before, tokens, window, sinks
    (1, 1, 64, 0, 1, 0, 0), (4, 2, 64, 100, 1, 0, 0), (40, 8, 128, 1000, 1, 0, 0), (32, 16, 128, 63, 1, 0, 0), (8, 1, 128, 64, 1, 0, 0),
    (6, 6, 80, 129, 1, 0, 0), (5, 1, 96, 257, 1, 0, 0), (16, 2, 256, 300, 1, 0, 0), (17, 1, 64, 90, 1, 0, 0), (32, 1, 256, 70, 1, 0, 0),
    (64, 1, 128, 200, 1, 0, 0), (48, 1, 192, 130, 1, 0, 0), (2, 1, 20, 40, 1, 0, 0), (3, 3, 1, 5, 1, 0, 0), (4, 4, 130, 66, 1, 0, 0),
    (4, 2, 64, 700, 1, 100, 0), (4, 2, 64, 700, 1, 100, 4), (10, 2, 128, 1500, 1, 64, 64), (4, 1, 64, 700, 1, 1, 0), (4, 1, 64, 700, 1, 1, 130),
    (4, 1, 64, 300, 1, 1000, 4), (8, 2, 64, 500, 1, 5, 2**31 - 1), (4, 2, 64, 190, 1, 2**31 - 1, 0),
    (40, 8, 128, 500, 2, 0, 0), (4, 2, 64, 61, 5, 0, 0), (10, 2, 64, 100, 7, 33, 3), (4, 1, 128, 0, 33, 0, 0), (8, 2, 128, 0, 64, 0, 0),
    (4, 2, 128, 0, 129, 0, 0), (5, 1, 128, 0, 301, 0, 0), (8, 8, 64, 37, 200, 0, 0), (4, 1, 256, 10, 150, 0, 0), (3, 1, 96, 1, 190, 0, 0),
    (12, 2, 80, 100, 130, 50, 0), (4, 2, 128, 600, 130, 64, 4), (4, 1, 64, 1000, 300, 128, 65), (2, 1, 32, 500, 260, 1, 1), (6, 1, 192, 64, 128, 0, 0),
]


def _attend_case(lane, heads, kv, width, before, n, window, sinks, seed, scale=None, sharp=1.0):
    rng = _rng(8, seed)
    total = before + n
    k, v, q = _values(rng, total, kv, width), _values(rng, total, kv, width), _values(rng, n, heads, width) * np.float32(sharp)
    with QuantizedKvCache(lane, 1, 1, kv, width, total) as cache:
        _put(lane, cache, 0, k[None], v[None])
        cache.set_lengths([before])
        qb = lane.upload_raw(q)
        guard = lane.upload_raw(np.full(n * heads * width + 64, 3.0, np.float32))
        cache.attention(0, qb, heads, n, window=window, sinks=sinks, scale=scale, out=guard)
        got = lane.read(guard)
        assert np.all(got[n * heads * width:] == 3.0)
        got = got[:n * heads * width].reshape(n, heads, width)
        kq, vq = ref.cached(k), ref.cached(v)
        want, reach = ref.attend(q, kq, vq, before, window, sinks, scale)
        qb.dispose()
        guard.dispose()
    return got, want, _tolerance(reach, total, width, np.abs(vq).max())


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_attention_against_64_bits(lane, case):
    got, want, tolerance = _attend_case(lane, *case, seed=CASES.index(case))
    assert np.isfinite(got).all()
    assert np.abs(got - want).max() <= tolerance, (np.abs(got - want).max(), tolerance)
    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)


@pytest.mark.parametrize("case", [(4, 1, 64, 3000, 1, 0, 0), (6, 2, 80, 2500, 3, 0, 0), (2, 1, 256, 2700, 1, 0, 0), (8, 1, 64, 6000, 40, 0, 0),
                                  (3, 1, 128, 900, 50, 700, 5), (5, 1, 96, 640, 1, 0, 0), (2, 2, 192, 700, 70, 0, 0), (4, 1, 32, 2100, 33, 0, 0)],
                         ids=lambda c: "-".join(map(str, c)))
def test_long_spans_in_parts(lane, case):
    """Spans of a few and of many parts, whose partial results are added up in two ways."""
    got, want, tolerance = _attend_case(lane, *case, seed=63)
    assert np.abs(got - want).max() <= tolerance, (np.abs(got - want).max(), tolerance)
    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)


@pytest.mark.parametrize("heads,kv,n", [(4, 2, 1), (4, 1, 200)])
def test_sharp_flat_and_zero_scales(lane, heads, kv, n):
    for scale, sharp in ((None, 12.0), (0.0, 1.0), (1e-30, 1.0), (1.0, 1e-20), (None, 1e-30), (1e-18, 1e18)):
        got, want, tolerance = _attend_case(lane, heads, kv, 64, 200, n, 0, 0, 99, scale, sharp)
        assert np.isfinite(got).all() and np.abs(got - want).max() <= tolerance, (scale, sharp)


@pytest.mark.parametrize("n", [1, 150])
def test_a_long_tail_of_small_probabilities_is_not_lost(lane, n):
    """One key 17 above all others: every other probability is 4e-8, together they are a visible share."""
    width, before = 64, 20000
    k, v = np.zeros((before + n, 1, width), np.float32), np.zeros((before + n, 1, width), np.float32)
    k[0, 0, 0], v[:, 0, 1], v[0, 0, 1], v[0, 0, 0] = 17.0, 1.0, 0.0, 1.0
    q = np.zeros((n, 1, width), np.float32)
    q[..., 0] = 1.0
    with QuantizedKvCache(lane, 1, 1, 1, width, before + n) as cache:
        _put(lane, cache, 0, k[None], v[None])
        cache.set_lengths([before])
        qb = lane.upload_raw(q)
        out = cache.attention(0, qb, 1, n, scale=1.0)
        got = lane.read(out).reshape(n, width)
    others = (before + np.arange(n)) * np.exp(-17.0)
    # relative error: exp at -17 (25 * 2^-24), two parts of a probability (2^-21), an FP32 sum of up to 20140 equal terms one
    # after the other (20140 * 2^-24 = 1.2e-3, which the order of the terms decides); a lost tail would be off by 1
    bound = (25 + 8 + before + n) * 2.0 ** -24
    assert np.abs(got[:, 1] / (others / (1 + others)) - 1).max() < bound
    for b in (qb, out):
        b.dispose()


@pytest.mark.parametrize("n", [1, 140])
def test_hidden_keys_have_no_influence(lane, n):
    """Blocks and tokens a row does not see may hold anything, NaN scales too; what it sees makes it NaN."""
    heads, kv, width, before, window, sinks = 4, 2, 64, 320, 100, 4
    rng = _rng(9, n)
    k, v, q = _values(rng, before + n, kv, width), _values(rng, before + n, kv, width), _values(rng, n, heads, width)
    k[128, 0, 0], v[129, 1, 3] = np.nan, np.inf                     # block 2: tokens 128 .. 191
    with QuantizedKvCache(lane, 1, 1, kv, width, before + n + 64) as cache:
        _put(lane, cache, 0, k[None], v[None])
        cache.set_lengths([before])
        qb = lane.upload_raw(q)
        out = cache.attention(0, qb, heads, n, window=window, sinks=sinks)
        got = lane.read(out).reshape(n, heads, width)
        clean_k, clean_v = k.copy(), v.copy()
        clean_k[128:192], clean_v[128:192] = 0.0, 0.0
        kq, vq = ref.cached(clean_k), ref.cached(clean_v)
        want, reach = ref.attend(q, kq, vq, before, window, sinks)
        p = before + np.arange(n)
        sees = (p - window + 1 <= 191)[:, None] & np.ones(heads, bool)
        assert np.isnan(got[sees]).all()
        assert np.isfinite(got[~sees]).all()
        assert np.abs(got - want)[~sees].max() <= _tolerance(reach, before + n, width, np.abs(vq).max())
        # a query that is not finite: its own rows alone
        q[0, 1, 5] = np.inf
        lane.write(qb, q)
        cache.attention(0, qb, heads, n, window=window, sinks=sinks, out=out)
        again = lane.read(out).reshape(n, heads, width)
        assert np.isnan(again[0, 1]).all()
        keep = np.ones((n, heads), bool)
        keep[0, 1] = False
        assert np.array_equal(again[keep], got[keep], equal_nan=True)
        for b in (qb, out):
            b.dispose()


@pytest.mark.parametrize("n,heads", [(1, 8), (3, 8), (90, 4)])
def test_sequences_of_a_batch_do_not_influence_each_other(lane, n, heads):
    B, kv, width = 5, 2, 128
    before = np.array([0, 700, 64, 1, 333], np.int32)
    counts = np.array([n, max(1, n // 2), n, 1, n], np.int32)
    rng = _rng(10, n)
    total = int(before.max()) + n
    k, v, q = (_values(rng, B * m, h, width).reshape(B, m, h, width) for m, h in ((total, kv), (total, kv), (n, heads)))
    with QuantizedKvCache(lane, 1, B, kv, width, total) as cache, QuantizedKvCache(lane, 1, 1, kv, width, total) as single:
        cb = lane.upload_raw(before + counts)
        _put(lane, cache, 0, k, v, counts=cb)
        cache.set_lengths(before)
        lane.write(cb, counts)
        qb, out = lane.upload_raw(q), lane.upload_raw(np.zeros_like(q))
        cache.attention(0, qb, heads, n, counts=cb, window=200, sinks=2, out=out)
        got = lane.read(out).reshape(q.shape)
        cache.attention(0, qb, heads, n, counts=cb, window=200, sinks=2, out=out)
        assert np.array_equal(got, lane.read(out).reshape(q.shape))             # the same on every run
        for b in range(B):
            c, t = int(counts[b]), int(before[b] + counts[b])
            kq, vq = ref.cached(k[b, :t]), ref.cached(v[b, :t])
            want, reach = ref.attend(q[b, :c], kq, vq, int(before[b]), 200, 2)
            assert np.abs(got[b, :c] - want).max() <= _tolerance(reach, t, width, np.abs(vq).max())
            assert not got[b, c:].any()
        for x in (cb, qb, out):
            x.dispose()


@pytest.mark.parametrize("width,window,sinks", [(32, 0, 0), (64, 30, 2), (96, 0, 0), (128, 70, 1), (192, 0, 0)])
@pytest.mark.parametrize("sequences", [40, 65])
def test_many_pairs_of_a_few_rows(lane, sequences, width, window, sinks):
    """More row tiles than compute units: the forms of the prompt kernel that long prompts of many heads take."""
    kv, heads, n, before = 8, 8, 37, 100
    rng = _rng(62, sequences, width)
    k, v = (rng.standard_normal((sequences, before + n, kv, width)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((sequences, n, heads, width)).astype(np.float32)
    counts = rng.integers(0, n + 1, sequences).astype(np.int32)
    counts[:2] = n, 1
    with QuantizedKvCache(lane, 1, sequences, kv, width, before + n) as cache:
        _put(lane, cache, 0, k, v)
        cache.set_lengths([before] * sequences)
        qb, cb, out = lane.upload_raw(q), lane.upload_raw(counts), lane.upload_raw(np.full(q.size, 7.0, np.float32))
        cache.attention(0, qb, heads, n, window=window, sinks=sinks, counts=cb, out=out)
        got = lane.read(out).reshape(q.shape)
        for b in list(range(0, sequences, 9)) + [1]:
            c = int(counts[b])
            kb, vb = ref.cached(k[b]), ref.cached(v[b])
            if c:
                want, reach = ref.attend(q[b, :c], kb, vb, before, window, sinks)
                assert np.abs(got[b, :c] - want).max() <= _tolerance(reach, before + n, width, np.abs(vb).max()), b
            assert np.all(got[b, c:] == 7.0)
        for b in (qb, cb, out):
            b.dispose()


def test_attention_far_behind_four_gigabytes(lane):
    """One head of 256 components and 18 million tokens: the codes of its last blocks lie behind 2^32 bytes."""
    width, capacity = 256, 18 << 20
    rng = _rng(11)
    n = 200
    first = capacity - 256
    k, v, q = (_values(rng, n, 1, width) for _ in range(3))
    with QuantizedKvCache(lane, 1, 1, 1, width, capacity) as cache:
        cache.set_lengths([first])
        _put(lane, cache, 0, k[None], v[None])
        got_k, got_v = _read(lane, cache, 0, n, first=[first])
        assert np.array_equal(got_k[0], ref.cached(k)) and np.array_equal(got_v[0], ref.cached(v))
        qb = lane.upload_raw(q)
        for rows, at in ((1, n - 1), (100, n - 100)):               # a window that stays inside what was stored
            cache.set_lengths([first + at])
            part = Rows(qb, width, 0, at * width)
            out = cache.attention(0, part, 1, rows, window=90)
            got = lane.read(out).reshape(rows, 1, width)
            want, reach = ref.attend(q[at:], got_k[0], got_v[0], at, 90)
            assert np.abs(got - want).max() <= _tolerance(reach, n, width, np.abs(got_v).max())
            out.dispose()
        qb.dispose()
    lane.trim()


def test_one_captured_step_serves_every_length(lane):
    """store -> attention -> advance in a graph, replayed token by token with eager work in between, against the eager steps."""
    layers, B, kv, heads, width, steps = 2, 2, 2, 8, 64, 70
    rng = _rng(12)
    k, v = (_values(rng, B * steps, kv, width).reshape(steps, B, 1, kv, width) for _ in range(2))
    q = _values(rng, B * steps, heads, width).reshape(steps, B, 1, heads, width)
    freq = lane.upload_raw(Rotary.frequencies(width))
    rot = Rotary(freq, width)
    start = np.array([0, 30], np.int32)

    with QuantizedKvCache(lane, layers, B, kv, width, 200) as cache:
        lead = _values(rng, B * 30, kv, width).reshape(B, 30, kv, width)
        kb, vb, qb = lane.upload_raw(k[0]), lane.upload_raw(v[0]), lane.upload_raw(q[0])
        turned, out = lane.allocate(q[0].size), lane.allocate(q[0].size)

        def fresh():
            cache.reset()
            for layer in range(layers):
                _put(lane, cache, layer, lead, lead, rotary=rot)
            cache.set_lengths(start)

        def step():
            for layer in range(layers):
                cache.store(layer, kb, vb, 1, rotary=rot, q=qb, q_out=turned, heads=heads)
                cache.attention(layer, turned, heads, 1, window=50, sinks=3, out=out)
            cache.advance(1)

        def run(do):
            got = []
            for s in range(steps):
                for buf, x in ((kb, k), (vb, v), (qb, q)):
                    lane.write(buf, x[s])
                do()
                got.append(lane.read(out))
            return np.stack(got), cache.read_lengths()

        fresh()
        eager, lengths = run(step)
        assert list(lengths) == [steps, 30 + steps] and np.isfinite(eager).all()
        fresh()
        lane.graph_begin()
        step()
        graph = lane.graph_end()
        assert list(cache.read_lengths()) == list(start)            # (recorded, not run)
        replayed, lengths = run(lambda: lane.graph_launch(graph))
        assert np.array_equal(eager, replayed) and list(lengths) == [steps, 30 + steps]
        lane.graph_destroy(graph)
        for x in (kb, vb, qb, turned, out, freq):
            x.dispose()


def test_graphs_and_eager_calls_share_the_scratch_memory():
    """Long caches leave partial results in the lane's scratch block: two graphs and eager work in turn, two layers each."""
    kv, heads, width, before = 2, 8, 128, 9000
    rng = _rng(13)
    k, v = (_values(rng, 2 * (before + 5), kv, width).reshape(2, 1, before + 5, kv, width) for _ in range(2))
    with HipExecutionLane(0) as lane, QuantizedKvCache(lane, 2, 1, kv, width, before + 5) as cache:
        for layer in range(2):
            _put(lane, cache, layer, k[layer], v[layer])
        cache.set_lengths([before])
        qb = [lane.upload_raw(_values(rng, n, heads, width)) for n in (1, 5, 40)]
        out = [[lane.allocate(n * heads * width) for _ in range(2)] for n in (1, 5, 40)]

        def step(which):
            n = (1, 5, 40)[which]
            for layer in range(2):
                cache.attention(layer, qb[which], heads, min(n, 5), out=out[which][layer])

        def results(which):
            step_out = [lane.read(b, np.uint32) for b in out[which]]
            for b in out[which]:
                lane.fill_u32(b, 0x7FC00000, b.nbytes // 4)
            return step_out

        # under capture the scratch block cannot come into being
        lane.graph_begin()
        cache.advance(1)
        with pytest.raises(NnHipError, match="before capturing"):
            step(0)
        lane.graph_destroy(lane.graph_end())
        eager = []
        for which in range(2):
            step(which)
            eager.append(results(which))
        graphs = []
        for which in range(2):
            lane.graph_begin()
            step(which)
            graphs.append(lane.graph_end())
        for which in (0, 1, 1, 0, 1, 0):
            lane.graph_launch(graphs[which])
            step(1 - which)                                             # eager work behind it, in the same scratch block
            for w in (which, 1 - which):
                for a, b in zip(results(w), eager[w]):
                    assert np.array_equal(a, b)
        # a larger call grows it; the graphs keep theirs
        with QuantizedKvCache(lane, 1, 64, 1, 256, 6000) as big:
            big.set_lengths([5000] * 64)
            x = lane.allocate(64 * 32 * 256)
            lane.fill_u32(x, 0, 64 * 32 * 256)
            big.store(0, x, x, 1)
            big.attention(0, x, 32, out=lane.allocate(64 * 32 * 256))
            lane.synchronize()
        for which in (1, 0):
            lane.graph_launch(graphs[which])
            for a, b in zip(results(which), eager[which]):
                assert np.array_equal(a, b)
        for g in graphs:
            lane.graph_destroy(g)


def test_refusals(lane):
    with QuantizedKvCache(lane, 1, 2, 2, 64, 100) as cache:
        small, big = lane.allocate(16), lane.allocate(4 * 2 * 4 * 64)
        freq = lane.upload_raw(Rotary.frequencies(64))
        for call in (lambda: cache.store(0, small, big), lambda: cache.store(0, big, big, 0), lambda: cache.store(0, big, big, heads=4),
                     lambda: cache.store(0, big, big, q=big, heads=4), lambda: cache.store(0, big, big, rotary=Rotary(freq, 128)),
                     lambda: cache.store(0, big, big, counts=lane.allocate_bytes(4)),
                     lambda: cache.attention(0, big, 3), lambda: cache.attention(0, big, 4, window=-1), lambda: cache.attention(0, big, 4, sinks=-1),
                     lambda: cache.attention(0, big, 4, scale=float("nan")), lambda: cache.attention(0, big, 4, scale=-1.0),
                     lambda: cache.attention(0, big, 4, out=small), lambda: cache.read(0, 1), lambda: cache.read(0, 0, k_out=big),
                     lambda: cache.set_lengths([1]), lambda: cache.set_lengths([1, 101]), lambda: cache.set_lengths([-1, 0]),
                     lambda: Rows(big, -1), lambda: Rotary(freq, 63), lambda: Rotary(freq, 256), lambda: lane.wrap(0, 4)):
            with pytest.raises(ValueError):
                call()
        with pytest.raises(IndexError):
            cache.store(1, big, big)
        with pytest.raises(TypeError):
            cache.store(0, None, big)
        for call in (lambda: cache.attention(0, big, 4, out=big),                                  # in place
                     lambda: cache.attention(0, big, 4, out=Rows(big, 256, 0)),                    # sequences over each other
                     lambda: cache.advance(0)):
            with pytest.raises(NnHipError):
                call()
        with pytest.raises(NnHipError):
            QuantizedKvCache(lane, 1, 1, 1, 257, 10)
        with pytest.raises(ValueError):
            QuantizedKvCache(lane, 1, 0, 1, 64, 10)
        for b in (small, big, freq):
            b.dispose()
    with pytest.raises(ValueError):
        cache.reset()


def test_refusals_of_sizes_and_alignment(lane):
    """Counts beyond 32 bits in Python; addresses between FP32 values and positions near the largest integer in the C entry."""
    import ctypes
    from nntrain_amd import native
    lib, h = lane._lib, lane._handle
    with QuantizedKvCache(lane, 1, 2, 2, 64, 100) as cache:
        big, counts = lane.allocate(4 * 2 * 4 * 64), lane.allocate_bytes(16)
        off = counts.view(2, 12)
        still = Rows(big, 0, 0)
        for call in (lambda: cache.store(0, still, still, 2**31), lambda: cache.attention(0, still, 4, 2**31), lambda: cache.attention(0, still, 2**33),
                     lambda: cache.read(0, 2**31, k_out=still)):
            with pytest.raises(ValueError):
                call()
        freq = lane.upload_raw(Rotary.frequencies(64))
        for call in (lambda: cache.store(0, big, big, counts=off), lambda: cache.attention(0, big, 4, counts=off), lambda: cache.advance(1, counts=off),
                     lambda: cache.read(0, 1, first=off, k_out=big), lambda: cache.store(0, big, big, rotary=Rotary(freq.view(2, 128 - 4), 62))):
            with pytest.raises(NnHipError):
                call()
        size = ctypes.c_uint64()
        assert lib.nnhip_kv_cache_bytes(1, 1, 64, 2**30, ctypes.byref(size)) == 0 and lib.nnhip_kv_cache_bytes(1, 1, 64, 2**30 + 1, ctypes.byref(size)) != 0
        desc = native.KvCacheDesc(ctypes.sizeof(native.KvCacheDesc), 1, 1, 64, 2**30 + 1, 0, big.ptr, counts.ptr)
        assert lib.nnhip_kv_cache_advance(h, ctypes.byref(desc), 1, None) != 0
        for b in (big, counts, freq):
            b.dispose()


def test_native_refusals(lane):
    """What the C entry refuses by itself, without reaching a launch."""
    import ctypes
    from nntrain_amd import native
    lib, h = lane._lib, lane._handle
    data, lengths, rows = lane.allocate_bytes(1 << 20), lane.upload_raw(np.zeros(2, np.int32)), lane.allocate(4096)
    launches = lane.counters()["kernel_launches"]
    cache = dict(struct_size=ctypes.sizeof(native.KvCacheDesc), sequences=2, kv_heads=2, head_width=64, capacity=100, reserved=0,
                 data=data.ptr, lengths=lengths.ptr)
    r = native.RowsDesc(rows.ptr, 256, 512)
    store = dict(struct_size=ctypes.sizeof(native.KvStoreDesc), tokens=1, k=r, v=r)
    attend = dict(struct_size=ctypes.sizeof(native.AttentionDesc), tokens=1, q=native.RowsDesc(data.ptr, 256, 256), out=r, heads=4, scale=1.0)

    def status(fn, c, desc):
        return fn(h, ctypes.byref(native.KvCacheDesc(**c)), ctypes.byref(desc))

    for bad in (dict(struct_size=3), dict(sequences=0), dict(kv_heads=-1), dict(head_width=257), dict(capacity=0), dict(reserved=1),
                dict(data=None), dict(data=data.ptr + 4), dict(lengths=None)):
        assert status(lib.nnhip_kv_cache_store, {**cache, **bad}, native.KvStoreDesc(**store)) != 0, bad
        assert status(lib.nnhip_cached_attention, {**cache, **bad}, native.AttentionDesc(**attend)) != 0, bad
    for bad in (dict(struct_size=0), dict(tokens=0), dict(reserved=2), dict(heads=1), dict(q=r), dict(q_out=r), dict(rotary_width=64),
                dict(inv_freq=rows.ptr, rotary_width=63), dict(inv_freq=rows.ptr, rotary_width=66), dict(inv_freq=rows.ptr),
                dict(inv_freq=rows.ptr, rotary_width=64, rotary_style=2), dict(k=native.RowsDesc(None, 256, 512)),
                dict(k=native.RowsDesc(rows.ptr + 2, 256, 512)), dict(v=native.RowsDesc(rows.ptr, -1, 512)),
                dict(inv_freq=rows.ptr, rotary_width=64, q=r, q_out=native.RowsDesc(rows.ptr, 256, 1024), heads=4)):
        assert status(lib.nnhip_kv_cache_store, cache, native.KvStoreDesc(**{**store, **bad})) != 0, bad
    for bad in (dict(struct_size=0), dict(tokens=0), dict(heads=3), dict(heads=0), dict(window=-1), dict(sinks=-1), dict(scale=float("inf")),
                dict(q=r), dict(out=native.RowsDesc(rows.ptr, 256, 0))):
        assert status(lib.nnhip_cached_attention, cache, native.AttentionDesc(**{**attend, **bad})) != 0, bad
    assert lib.nnhip_kv_cache_store(h, None, None) != 0 and lib.nnhip_cached_attention(h, None, None) != 0
    with pytest.raises(NnHipError):
        check(lib.nnhip_kv_cache_advance(None, None, 1, None), "kv_cache_advance")
    assert lane.counters()["kernel_launches"] == launches
    for b in (data, lengths, rows):
        b.dispose()


@pytest.mark.parametrize("n,heads", [(2, 1), (6, 4), (20, 2), (150, 4), (300, 1)])
@pytest.mark.parametrize("size", [1e6, 1e12, 1e30])
def test_large_values_of_hidden_blocks_have_no_influence(lane, n, heads, size):
    """Rows that are worked on side by side: the first ones still see a block of very large values, or see one already that
    begins behind the others.  Those that do not keep their accuracy."""
    kv, width = 1, 64
    for window, before, block in ((64, 126, 0), (64, 127, 2), (320, 382, 0), (320, 383, 6)):
        rng = _rng(15, n, heads, block)
        k, v, q = _values(rng, before + n, kv, width), _values(rng, before + n, kv, width), _values(rng, n, heads, width)
        v[64 * block:64 * block + 64] *= np.float32(size)
        with QuantizedKvCache(lane, 1, 1, kv, width, before + n) as cache:
            _put(lane, cache, 0, k[None], v[None])
            cache.set_lengths([before])
            qb = lane.upload_raw(q)
            out = cache.attention(0, qb, heads, n, window=window)
            got = lane.read(out).reshape(n, heads, width)
            for b in (qb, out):
                b.dispose()
        kq, vq = ref.cached(k), ref.cached(v)
        want, reach = ref.attend(q, kq, vq, before, window)
        p = before + np.arange(n)
        sees = (p >= 64 * block) & (p - window + 1 < 64 * block + 64)
        others = np.delete(vq, np.s_[64 * block:64 * block + 64], 0)
        assert sees.any() and not sees.all()
        assert np.abs(got - want)[~sees].max() <= _tolerance(reach, before + n, width, np.abs(others).max())
        assert np.abs(got - want)[sees].max() <= _tolerance(reach, before + n, width, np.abs(vq).max())


@pytest.mark.parametrize("pieces", [[13], [12, 1], [5, 8], [1] * 13, [3, 10], [13 + 3, 1]])
def test_turned_keys_do_not_depend_on_how_the_tokens_arrive(lane, pieces):
    """A key one of whose components lies within 2^-49 of the border between two FP32 numbers after its turn (token 6412, angle
    6412 * 0.9): the same number whichever call brings the token, and with it the same scale of the block."""
    width, start = 32, 6400
    k = np.zeros((1, sum(pieces), 1, width), np.float32)
    k[0, 12, 0, 0] = 1.2270393371582031
    freq = lane.upload_raw(np.array([0.9], np.float32))
    with QuantizedKvCache(lane, 1, 1, 1, width, start + k.shape[1]) as cache:
        def stored(parts):
            cache.set_lengths([start])
            at = 0
            for p in parts:
                _put(lane, cache, 0, k[:, at:at + p], k[:, at:at + p], rotary=Rotary(freq, 2))
                cache.advance(p)
                at += p
            return _read(lane, cache, 0, at, first=[start])[0][0, 12, 0]
        got, whole = stored(pieces), stored([sum(pieces)])
        assert np.array_equal(got, whole) and abs(got[0] / (1.2270393371582031 * np.cos(6412 * np.float64(np.float32(0.9)))) - 1) < 2.0 ** -22
    freq.dispose()


def test_refusals_of_launches_of_too_many_threads(lane):
    """A launch holds fewer than 2^32 threads: what would need more is refused before it is tried (8: too large)."""
    import ctypes
    from nntrain_amd import native
    lib, h = lane._lib, lane._handle
    with QuantizedKvCache(lane, 1, 1, 1, 1, 100) as cache:
        lane.write(cache.lengths, np.array([-1], np.int32))             # (left out, whatever is asked for)
        one = lane.allocate(4)
        still = native.RowsDesc(one.ptr, 0, 0)
        launches = lane.counters()["kernel_launches"]
        store = native.KvStoreDesc(struct_size=ctypes.sizeof(native.KvStoreDesc), tokens=2**30, k=still, v=still)
        assert lib.nnhip_kv_cache_store(h, cache._refs[0], ctypes.byref(store)) == 8
        far = native.RowsDesc(one.ptr, 1, 2**30)
        assert lib.nnhip_kv_cache_read(h, cache._refs[0], None, 2**30, ctypes.byref(far), None) == 8
        many = native.KvCacheDesc(ctypes.sizeof(native.KvCacheDesc), 2**22, 1, 1, 100, 0, one.ptr, cache.lengths.ptr)
        attend = native.AttentionDesc(struct_size=ctypes.sizeof(native.AttentionDesc), tokens=200, q=still, out=native.RowsDesc(one.ptr + 4, 1, 200),
                                      heads=1, scale=1.0)
        assert lib.nnhip_cached_attention(h, ctypes.byref(many), ctypes.byref(attend)) == 8
        assert lane.counters()["kernel_launches"] == launches
        one.dispose()


def test_tokens_behind_a_row_act_through_the_scale_of_its_block_alone(lane):
    """A call stores its tokens before it attends: a row reads what the cache then stands for, later tokens in the scale."""
    kv, heads, width, n = 1, 2, 64, 10
    rng = _rng(16)
    k, v, q = _values(rng, n, kv, width), _values(rng, n, kv, width), _values(rng, n, heads, width)
    for size in (30.0, 1000.0, np.inf):
        late_k, late_v = k.copy(), v.copy()
        late_k[n - 1], late_v[n - 1] = size, size
        with QuantizedKvCache(lane, 1, 1, kv, width, n) as cache:
            _put(lane, cache, 0, late_k[None], late_v[None])
            qb = lane.upload_raw(q)
            out = cache.attention(0, qb, heads, n)
            together = lane.read(out).reshape(n, heads, width)
            kq, vq = ref.cached(late_k), ref.cached(late_v)
            if np.isfinite(size):
                want, reach = ref.attend(q, kq, vq, 0)
                assert np.abs(together - want)[:n - 1].max() <= _tolerance(reach, n, width, np.abs(vq[:n - 1]).max() + np.abs(vq).max() / 127)
            else:
                assert np.isnan(together).all()
            # token by token nothing behind a row has any influence
            cache.reset()
            for i in range(n - 1):
                _put(lane, cache, 0, late_k[None, i:i + 1], late_v[None, i:i + 1])
                part = Rows(qb, heads * width, 0, i * heads * width)
                one = cache.attention(0, part, heads)
                want, reach = ref.attend(q[i:i + 1], ref.cached(k[:i + 1]), ref.cached(v[:i + 1]), i)
                assert np.abs(lane.read(one).reshape(1, heads, width) - want).max() <= _tolerance(reach, i + 1, width, np.abs(v[:i + 1]).max())
                cache.advance(1)
                one.dispose()
            for b in (qb, out):
                b.dispose()


@pytest.mark.parametrize("n", [1, 50, 1100])
def test_a_tail_far_below_one_key_over_a_long_cache(lane, n):
    """One key 17 or 21.6 above 30000 others: what a block adds is a few or less than one of the large sum's last places.  Bar:
    (n / 16) 2^-23 of the sums, numerator and denominator, and the parts of a probability."""
    width, heads, before = 64, 8, 30000
    for gap in (17.0, 21.6):
        k, v = (np.zeros((before + n, heads, width), np.float32) for _ in range(2))
        k[0, :, 0], v[1:, :, 1], v[0, :, 0] = gap, 1.0, 1.0
        q = np.zeros((n, heads, width), np.float32)
        q[..., 0] = 1.0
        with QuantizedKvCache(lane, 1, 1, heads, width, before + n) as cache:
            _put(lane, cache, 0, k[None], v[None])
            cache.set_lengths([before])
            qb = lane.upload_raw(q)
            out = cache.attention(0, qb, heads, n, scale=1.0)
            got = lane.read(out).reshape(n, heads, width)
            for b in (qb, out):
                b.dispose()
        others = ((before + np.arange(n)) * np.exp(-float(np.float32(gap / 127) * np.float32(127))))[:, None]
        bar = 2 * ((before + n) / 16 * 2.0 ** -23 + 2.0 ** -21)
        assert np.abs(got[..., 1] - others / (1 + others)).max() <= bar and np.abs(got[..., 0] - 1 / (1 + others)).max() <= bar
        assert not got[..., 2:].any()
