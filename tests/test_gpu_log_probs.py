"""Token log probabilities, entropy and top alternatives, through the package, against 64-bit numpy.

Bars: a term e^(x - m) is off by (|x - m| * 1.45 + 3) * 2^-24 of itself (argument, constant and exponential), sums are 64-bit, so ln S is
off by at most that factor at the largest |x - m| that matters; with |x - m| < 90 for every term that is not zero: 2^-17.
A log probability has that error plus one rounding; T / S and ln S have it relative to themselves (all terms of one sign).
"""
import numpy as np
import pytest

import kv_reference as ref
from nntrain_amd import HipExecutionLane, qwen35_gpu
from nntrain_amd.native import LogProbsDesc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lane():
    with HipExecutionLane(0) as ln:
        yield ln


def _run(lane, x, targets=None, top=0, stride=None, **kw):
    rows, vocabulary = x.shape
    stride = vocabulary if stride is None else stride
    padded = np.full(((rows - 1) * stride + vocabulary,), np.nan, np.float32)
    for r in range(rows):
        padded[r * stride:r * stride + vocabulary] = x[r]
    xb = lane.upload_raw(padded)
    tb = lane.upload_raw(np.asarray(targets, np.int32)) if targets is not None else None
    got = qwen35_gpu.token_log_probs(lane, xb, rows, vocabulary, tb, top, stride, **kw)
    out = [lane.read(b, t, rows * m).reshape(rows, m) if b is not None else None
           for b, t, m in zip(got, (np.float32, np.float32, np.int32, np.float32), (1, 1, top, top))]
    for b in (xb, tb, *got):
        if b is not None:
            b.dispose()
    return out


def _order(x):
    v = np.where(np.isnan(x), np.inf, x)
    return np.argsort(-v, axis=1, kind="stable")


def _check(lane, x, targets, top, stride=None):
    lp, entropy, ids, top_lp = _run(lane, x, targets, top, stride)
    want, want_entropy = ref.log_probs(x)
    at = want[np.arange(x.shape[0]), targets]
    tolerance = 2.0 ** -17 * np.minimum(1.0, np.exp(0)) + 2.0 ** -23 * np.abs(at)
    assert np.all(np.abs(lp[:, 0] - at) <= tolerance) and np.all(np.abs(lp[:, 0] - at) <= 1e-5 * np.abs(at) + 2e-6)
    assert np.all(np.abs(entropy[:, 0] - want_entropy) <= 2.0 ** -16 * want_entropy)
    if top:
        order = _order(x)[:, :top]
        assert np.array_equal(ids, order)
        at = np.take_along_axis(want, order.astype(np.int64), 1)
        fine = np.isfinite(at)
        assert np.array_equal(fine, np.isfinite(top_lp)) and np.all(np.abs(top_lp - at)[fine] <= 2e-6 + 1e-5 * np.abs(at[fine]))


@pytest.mark.parametrize("rows,vocabulary,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 63, 5), (5, 64, 64), (4, 65, 20), (1, 320, 1), (3, 1023, 7),
                                                 (2, 4096, 32), (1, 4097, 64), (1, 32000, 1), (7, 32001, 20), (33, 5000, 3), (2, 151937, 40), (1, 262144, 64),
                                                 (300, 1500, 5), (2100, 70, 2)])
def test_random_rows(lane, rows, vocabulary, top):
    rng = np.random.default_rng([rows, vocabulary])
    x = (rng.standard_normal((rows, vocabulary)) * 3).astype(np.float32)
    _check(lane, x, rng.integers(0, vocabulary, rows), top)
    if vocabulary > 8:
        _check(lane, x, rng.integers(0, vocabulary, rows), top, stride=vocabulary + 3)


@pytest.mark.parametrize("vocabulary", [300, 40000])
def test_equal_rising_and_falling_logits(lane, vocabulary):
    i = np.arange(vocabulary)
    x = np.stack([np.zeros(vocabulary), i * 1e-4, -i * 1e-4, (i % 7).astype(float), np.where(i % 2 == 0, -0.0, 0.0),
                  np.where(i == vocabulary - 1, 5.0, 1.0)]).astype(np.float32)
    _check(lane, x, np.array([0, 5, 7, 3, 2, vocabulary - 1]), 64)


@pytest.mark.parametrize("rows,vocabulary,top", [(1, 3000, 64), (300, 3000, 64), (3, 1500, 5), (2, 70000, 33), (300, 20000, 20), (1, 16384, 16)])
def test_many_equal_logits_and_few_finite_ones(lane, rows, vocabulary, top):
    """More logits at the threshold than any list holds, rows with fewer finite logits than alternatives, and ties between pieces."""
    rng = np.random.default_rng([77, rows, vocabulary])
    x = rng.integers(0, 3, (rows, vocabulary)).astype(np.float32)
    x[0, : vocabulary // 2] = -np.inf
    if rows > 1:
        x[1] = -np.inf
        x[1, rng.choice(vocabulary, top - 2, replace=False)] = rng.standard_normal(top - 2)
        x[rows - 1] = np.sort(rng.standard_normal(vocabulary)).astype(np.float32)
    buffer = lane.upload_raw(x)
    got = qwen35_gpu.token_log_probs(lane, buffer, rows, vocabulary, top=top)
    ids, lps = lane.read(got.top_ids, np.int32).reshape(rows, top), lane.read(got.top_log_probs).reshape(rows, top)
    want, _ = ref.log_probs(x)
    for r in range(rows):
        order = np.argsort(-x[r], kind="stable")[:top]
        assert np.array_equal(ids[r], order), r
        expected = want[r, order]
        finite = np.isfinite(expected)
        assert np.array_equal(finite, np.isfinite(lps[r]))
        # the logarithm of a sum of at most 2^24 exponentials, each within 2^-22 of its own, in 64 bits, and one rounding
        assert np.abs(lps[r][finite] - expected[finite]).max() <= 2.0 ** -21 + 2.0 ** -24 * np.abs(expected[finite]).max()
    for b in (buffer, got.entropy, got.top_ids, got.top_log_probs):
        b.dispose()


def test_near_certain_rows_keep_their_digits(lane):
    """The largest logit 10 .. 80 above the others: ln p of it and the entropy are tiny and relative accuracy counts."""
    vocabulary = 5000
    x = np.zeros((8, vocabulary), np.float32)
    gaps = np.arange(10, 90, 10)
    x[np.arange(8), 100 + gaps] = gaps
    lp, entropy, ids, top_lp = _run(lane, x, 100 + gaps, 1)
    rest = (vocabulary - 1) * np.exp(-gaps.astype(np.float64))
    want = -np.log1p(rest)
    want_entropy = np.log1p(rest) + rest * gaps / (1 + rest)
    # one term e^-gap: (80 * 1.45 + 3) * 2^-24 = 7.1e-6 of itself; S is a 64-bit sum: below rest = 1e-16 * 2^-? nothing is left of it
    fine = rest > 1e-9
    assert np.abs(lp[fine, 0] / want[fine] - 1).max() < 1e-5 and np.abs(entropy[fine, 0] / want_entropy[fine] - 1).max() < 1e-5
    assert np.abs(lp[:, 0] - want).max() < 1e-5 * np.abs(want).max() and np.all(lp <= 0) and np.all(entropy >= 0)
    assert np.array_equal(ids[:, 0], 100 + gaps) and np.array_equal(top_lp, lp)


def test_masked_and_undefined_rows(lane):
    vocabulary = 9000
    rng = np.random.default_rng(5)
    x = rng.standard_normal((8, vocabulary)).astype(np.float32)
    x[0, 10:] = -np.inf                                             # most of the vocabulary masked
    x[1] = -np.inf                                                  # everything masked
    x[2, 77] = np.inf
    x[3, 8999] = np.nan
    x[4] = np.finfo(np.float32).min
    x[5, :] = -np.inf
    x[5, 4000] = -3.0
    x[6, 0] = -np.inf
    x[7] = np.where(np.arange(vocabulary) % 3 == 0, np.finfo(np.float32).max, -np.finfo(np.float32).max)
    targets = np.array([3, 0, 77, 0, 5, 4000, 0, 3])
    lp, entropy, ids, top_lp = _run(lane, x, targets, 20)
    assert np.array_equal(ids, _order(x)[:, :20])
    undefined = np.array([1, 2, 3])
    assert np.isnan(lp[undefined]).all() and np.isnan(entropy[undefined]).all() and np.isnan(top_lp[undefined]).all()
    want, want_entropy = ref.log_probs(x)
    for r in (0, 4, 5, 7):
        assert abs(lp[r, 0] - want[r, targets[r]]) < 1e-5 and abs(entropy[r, 0] - want_entropy[r]) < 1e-5 * max(1.0, want_entropy[r])
    assert lp[6, 0] == -np.inf and lp[5, 0] == 0.0 and entropy[5, 0] == 0.0
    assert np.all(top_lp[0, 10:] == -np.inf) and np.isfinite(top_lp[0, :10]).all()
    # targets outside the vocabulary
    lp, _, _, _ = _run(lane, x[:1].repeat(4, 0), [-1, vocabulary, 2**31 - 1, 4], 0)
    assert np.isnan(lp[:3]).all() and np.isfinite(lp[3])


def test_parts_that_are_not_asked_for_and_given_outputs(lane):
    x = np.random.default_rng(6).standard_normal((3, 777)).astype(np.float32)
    full = _run(lane, x, [1, 2, 3], 4)
    none = _run(lane, x, None, 4)
    assert none[0] is None and all(np.array_equal(a, b) for a, b in zip(none[1:], full[1:]))
    out = _run(lane, x, [1, 2, 3], 0)
    assert out[2] is None and np.array_equal(out[0], full[0]) and np.array_equal(out[1], full[1])
    ids = lane.upload_raw(np.full(3 * 4 + 5, -7, np.int32))
    xb = lane.upload_raw(x)
    qwen35_gpu.token_log_probs(lane, xb, 3, 777, None, 4, top_ids=ids)
    got = lane.read(ids, np.int32)
    assert np.array_equal(got[:12].reshape(3, 4), full[2]) and np.all(got[12:] == -7)
    for b in (ids, xb):
        b.dispose()


def test_replays_of_a_captured_call(lane):
    rows, vocabulary, top = 4, 50000, 8
    rng = np.random.default_rng(7)
    xb, tb = lane.allocate(rows * vocabulary), lane.upload_raw(np.arange(rows, dtype=np.int32))
    first = qwen35_gpu.token_log_probs(lane, xb, rows, vocabulary, tb, top)
    again = [lane.allocate_bytes(b.nbytes) for b in first]
    for b in qwen35_gpu.token_log_probs(lane, xb, rows, vocabulary, tb, top):
        b.dispose()
    lane.graph_begin()
    qwen35_gpu.token_log_probs(lane, xb, rows, vocabulary, tb, top, out=again[0], entropy=again[1], top_ids=again[2], top_log_probs=again[3])
    graph = lane.graph_end()
    for _ in range(4):
        lane.write(xb, (rng.standard_normal((rows, vocabulary)) * 4).astype(np.float32))
        qwen35_gpu.token_log_probs(lane, xb, rows, vocabulary, tb, top, out=first[0], entropy=first[1], top_ids=first[2], top_log_probs=first[3])
        lane.synchronize()
        lane.graph_launch(graph)
        for a, b in zip(first, again):
            assert np.array_equal(lane.read(a, np.uint32), lane.read(b, np.uint32))
    lane.graph_destroy(graph)
    for b in (xb, tb, *first, *again):
        b.dispose()


def test_refusals(lane):
    import ctypes
    x, t = lane.allocate(100), lane.upload_raw(np.zeros(2, np.int32))
    call = qwen35_gpu.token_log_probs
    for bad in (lambda: call(lane, x, 2, 51), lambda: call(lane, x, 0, 50), lambda: call(lane, x, 2, 0), lambda: call(lane, x, 2, 50, top=51),
                lambda: call(lane, x, 1, 100, top=65), lambda: call(lane, x, 2, 50, top=-1), lambda: call(lane, x, 2, 50, row_stride=49),
                lambda: call(lane, x, 4, 10, t), lambda: call(lane, x, 2, 50, out=x), lambda: call(lane, x, 2, 50, top_ids=t)):
        with pytest.raises(ValueError):
            bad()
    good = dict(struct_size=ctypes.sizeof(LogProbsDesc), rows=2, vocabulary=50, top=0, row_stride=50, logits=x.ptr, entropy=t.ptr)
    launches = lane.counters()["kernel_launches"]
    for bad in (dict(struct_size=1), dict(rows=0), dict(vocabulary=0), dict(logits=None), dict(row_stride=49), dict(top=2), dict(top=65, top_ids=t.ptr),
                dict(top_ids=t.ptr), dict(top_log_probs=t.ptr), dict(targets=t.ptr), dict(log_probs=t.ptr), dict(entropy=None), dict(rows=65536, row_stride=50)):
        assert lane._lib.nnhip_token_log_probs(lane._handle, ctypes.byref(LogProbsDesc(**{**good, **bad}))) != 0, bad
    assert lane._lib.nnhip_token_log_probs(lane._handle, None) != 0
    assert lane.counters()["kernel_launches"] == launches
    for b in (x, t):
        b.dispose()


def test_refusal_of_addresses_between_values(lane):
    import ctypes
    x = lane.allocate(200)
    good = dict(struct_size=ctypes.sizeof(LogProbsDesc), rows=2, vocabulary=50, top=1, row_stride=50, logits=x.ptr, targets=x.ptr, log_probs=x.ptr + 600,
                entropy=x.ptr + 620, top_ids=x.ptr + 640, top_log_probs=x.ptr + 660)
    launches = lane.counters()["kernel_launches"]
    for name in ("logits", "targets", "log_probs", "entropy", "top_ids", "top_log_probs"):
        assert lane._lib.nnhip_token_log_probs(lane._handle, ctypes.byref(LogProbsDesc(**{**good, name: good[name] + 2}))) != 0, name
    assert lane.counters()["kernel_launches"] == launches
    x.dispose()


@pytest.mark.parametrize("rows,vocabulary", [(1, 700), (3, 5000), (2, 40000), (300, 1200), (40, 262144)])
def test_near_certain_rows_keep_their_digits_down_to_the_least_exponential(lane, rows, vocabulary):
    """One logit 8 .. 87 above all others: ln p = -log1p(rest), rest = (V - 1) e^-gap, relative to itself however small.

    A term e^-gap is off by (gap * 1.45 + 3) * 2^-24 of itself (argument, constant, exponential), the sums are 64-bit, one rounding."""
    gaps = np.linspace(8, 87, rows).round()
    rng = np.random.default_rng([78, rows, vocabulary])
    at = rng.integers(0, vocabulary, rows)
    x = np.zeros((rows, vocabulary), np.float32)
    x[np.arange(rows), at] = gaps
    lp, entropy, ids, top_lp = _run(lane, x, at, 1)
    rest = (vocabulary - 1) * np.exp(-gaps)
    bar = (gaps * 1.45 + 3) * 2.0 ** -24 + 2.0 ** -24
    assert np.all(np.abs(lp[:, 0] / -np.log1p(rest) - 1) <= bar)
    assert np.all(np.abs(entropy[:, 0] / (np.log1p(rest) + rest * gaps / (1 + rest)) - 1) <= 2 * bar)
    assert np.array_equal(ids[:, 0], at) and np.array_equal(top_lp, lp)


@pytest.mark.parametrize("vocabulary", [64, 5000, 262144])
def test_rows_with_several_largest_logits(lane, vocabulary):
    """Equal largest logits, in one lane, in one wave and far apart: only one of them is left out of the rest."""
    x = np.full((4, vocabulary), -60.0, np.float32)
    places = [[0], [0, 1], [3, vocabulary - 1], [0, 7, 20, vocabulary // 2, vocabulary - 2, vocabulary - 1]]
    for r, p in enumerate(places):
        x[r, p] = 1.5
    lp, entropy, _, _ = _run(lane, x, [p[-1] for p in places], 0)
    for r, p in enumerate(places):
        rest = len(p) - 1 + (vocabulary - len(p)) * np.exp(-61.5)
        want, want_entropy = -np.log1p(rest), np.log1p(rest) + (vocabulary - len(p)) * np.exp(-61.5) * 61.5 / (1 + rest)
        assert abs(lp[r, 0] / want - 1) < 6e-6 and abs(entropy[r, 0] / want_entropy - 1) < 1.2e-5, r


@pytest.mark.parametrize("depth", [2.7, 12.1, 20.3, 31.7, 50.9, 70.3])
@pytest.mark.parametrize("vocabulary", [3000, 262144])
def test_flat_tails_far_below_the_largest_logit(lane, vocabulary, depth):
    """All logits but one the same far below it: what the exponential is off by does not average out.

    x - m is exact here (m = 0).  The power of two of the hardware is within 2^-23, the factor that makes up for the argument's
    rounding within 2^-24: 3 * 2^-24 of the rest; sixteen products with x - m meet in FP32: 16 * 2^-24 of T more; 2^-24 for the
    result's rounding."""
    depth = float(np.float32(depth))
    x = np.full((1, vocabulary), -depth, np.float32)
    x[0, 17] = 0.0
    lp, entropy, _, top_lp = _run(lane, x, [17], 2)
    rest = (vocabulary - 1) * np.exp(-depth)
    total = np.log1p(rest)
    assert abs(lp[0, 0] + total) <= 3 * 2.0 ** -24 * rest / (1 + rest) + 2.0 ** -24 * total
    want = total + depth * rest / (1 + rest)
    assert abs(entropy[0, 0] - want) <= 2.0 ** -24 * (3 * rest + 19 * depth * rest) / (1 + rest) + 2.0 ** -24 * want
    assert abs(top_lp[0, 1] + depth + total) <= 3 * 2.0 ** -24 * rest / (1 + rest) + 2.0 ** -24 * (depth + total)
