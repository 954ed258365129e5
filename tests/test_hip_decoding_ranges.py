"""GPU tests of the decoding operators over the ranges of their numbers: values of
keys side by side that are zero, tiny, far apart or near float32's largest, weights
that a long sum could lose, logits with offsets and at float32's lowest value.

Each call of more than eight rows of a key head runs in all of its forms: without a
workspace, with its keys split over blocks, and from packed tiles."""

from __future__ import annotations

import time

import numpy as np
import pytest

import decoding_cases as cases
from conftest import require_gpu

pytestmark = pytest.mark.gpu

EPS = cases.EPS


@pytest.fixture(scope="module")
def capi():
    require_gpu()
    import tensorcx_hip_capi
    assert tensorcx_hip_capi.available()
    return tensorcx_hip_capi


def f32(rng, *shape):
    return rng.normal(size=shape).astype(np.float32)


def window(capi, q, k, v, *, window=0, sinks=0, scale=None, lengths=None, workspace=True):
    """Outputs of (batch, heads, rows, features) arrays, with the workspace that is asked for or none."""
    dq, dk, dv = (capi.DeviceArray.from_numpy(x) for x in (q, k, v))
    out = capi.DeviceArray.from_numpy(np.full_like(q, 7))
    dn = None if lengths is None else capi.DeviceArray.from_numpy(np.asarray(lengths, np.int32))
    desc = capi.window_attention_desc(*q.shape[:2], k.shape[1], q.shape[2], k.shape[2], q.shape[3], window=window, sinks=sinks,
                                      scale=scale, lengths=None if dn is None else dn.ptr)
    ws = capi.window_attention_workspace(desc) if workspace else None
    capi.window_attention(dq.ptr, dk.ptr, dv.ptr, out.ptr, desc, workspace=ws)
    capi.synchronize()
    return out.numpy()


def cached(capi, q, keys, values, lengths, *, window=0, sinks=0, scale=None, workspace=True):
    dq, dk, dv, dn = (capi.DeviceArray.from_numpy(x) for x in (q, keys, values, np.asarray(lengths, np.int32)))
    out = capi.DeviceArray.from_numpy(np.full_like(q, 7))
    desc = capi.window_attention_desc(*q.shape[:2], keys.shape[1], q.shape[2], keys.shape[2], q.shape[3], window=window,
                                      sinks=sinks, scale=scale, lengths=dn.ptr)
    ws = capi.window_attention_workspace(desc, cache=True) if workspace else None
    capi.cache4_attention(dq.ptr, dk.ptr, dv.ptr, out.ptr, desc, workspace=ws)
    capi.synchronize()
    return out.numpy()


def check(out, q, k, v, lengths, window, sinks, scale, heads=None):
    """Against the plain form and its bound; of many heads those named."""
    share = q.shape[1] // k.shape[1]
    for b, h in heads or [(b, h) for b in range(q.shape[0]) for h in range(q.shape[1])]:
        key = np.s_[b:b + 1, h // share:h // share + 1]
        expected, bound = cases.attention(q[b:b + 1, h:h + 1], k[key], v[key], lengths[b:b + 1], window or None, sinks, scale)
        off = np.abs(out[b:b + 1, h:h + 1].astype(float) - expected)
        assert (off <= bound).all(), f"head {b}, {h}: off by up to {np.nanmax(off / np.maximum(bound, 1e-300)):.3g} of the bound"


# (batch, heads, kv_heads, rows, cols, features), with a workspace or not: the
# stream, 16 rows whole and over splits, packed tiles of every block size.
FORMS = [
    ((1, 2, 1, 2, 700, 64), True),
    ((1, 2, 1, 20, 200, 64), False),
    ((1, 2, 1, 20, 200, 128), False),
    ((1, 2, 1, 20, 900, 128), True),
    ((1, 1, 1, 1030, 1100, 64), True),
    ((43, 2, 2, 257, 260, 32), True),
    ((128, 1, 1, 257, 257, 80), True),
]


def form_heads(shape):
    batch, heads = shape[:2]
    return sorted({(0, 0), (batch // 2, heads - 1), (batch - 1, 0)})


# ------------------------------------------------------------------ values of keys
@pytest.mark.parametrize("far", [(0, 2.0 ** 60), (0, 1e20), (0, 1e30), (2.0 ** -70, 2.0 ** 76), (1.0, 2.0 ** 126), (0, 1e-30)],
                         ids=str)
@pytest.mark.parametrize("shape,workspace", FORMS, ids=str)
def test_values_far_apart(capi, shape, workspace, far):
    """Keys of one magnitude beside keys of another: a weight counts in the softmax's sum
    whatever its key's values are. (2^126 in one key alone, so that sums stay finite.)"""
    batch, heads, kv, rows, cols, d = shape
    rng = np.random.default_rng(61)
    q, k = f32(rng, batch, heads, rows, d), f32(rng, batch, kv, cols, d)
    v = np.sign(f32(rng, batch, kv, cols, d)) * np.float32(far[0])
    large = slice(1, None, 2) if far[1] < 1e36 else slice(1, 2)
    v[:, :, large] = np.abs(f32(rng, *v[:, :, large].shape)).clip(0.1, 2) * np.float32(far[1] / 2)
    for scale in (0.0, d ** -0.5):
        out = window(capi, q, k, v, scale=scale, workspace=workspace)
        check(out, q, k, v, [cols] * batch, 0, 0, scale, form_heads(shape))


@pytest.mark.parametrize("workspace", [False, True])
def test_small_weights_beside_a_huge_value(capi, workspace):
    """One key of values 2^126 and many of 1 whose weights are 2^-15 of its: together
    they are a quarter of the sum."""
    n, d = 8192, 16
    q, k, v = (np.zeros((1, 1, r, d), np.float32) for r in (16, n, n))
    q[..., 0], k[:, :, 0, 0], v[...] = 1, 15, 1
    v[:, :, 0] = 2.0 ** 126
    scale = float(np.float32(np.log(2)))
    out = window(capi, q, k, v, scale=scale, workspace=workspace)
    check(out, q, k, v, [n], 0, 0, scale)


def test_a_zero_valued_keys_weight(capi):
    """The weight of a key whose values are zero is as exact as that of any other.

    Two keys, of zeros and of ones, at scores of +a and -a in units of log2, a below 1 and of
    20 bits (held exactly): the output is w_b / (w_a + w_b). A score takes three roundings
    (the scale, log2 e, the product) of at most EPS, of both keys together 6 ln2 EPS of the
    quotient of the weights; the difference from the maximum, below 4, 4 ln2 EPS; two
    exponentials 4 EPS; the halves of w_b 4 EPS; the sum, its reciprocal and two products
    4 EPS: 19 EPS of the output."""
    rng = np.random.default_rng(62)
    d, scale = 16, float(np.float32(np.log(2)))
    q, k, v = (np.zeros((1, h, r, d), np.float32) for h, r in ((4096, 1), (1, 2), (1, 2)))
    q[..., 0] = rng.integers(1, 2 ** 20, q.shape[:3]) / 2 ** 20
    k[:, :, 0, 0], k[:, :, 1, 0], v[:, :, 1] = 1, -1, 1
    out = window(capi, q, k, v, scale=scale, workspace=False)
    s = q[..., :1].astype(float) * scale
    expected = np.exp(-s) / (np.exp(-s) + np.exp(s))
    assert (np.abs(out - expected) <= 19 * EPS * expected).all(), np.abs(out / expected - 1).max() / EPS


@pytest.mark.parametrize("rows", [16, 1030])
@pytest.mark.parametrize("workspace", [False, True])
def test_an_outlier_of_one_feature(capi, rows, workspace):
    """One feature of one key 2^18 above everything else, judged feature by feature.

    What the matrix form adds to a float32 kernel's error: weights are float16 halves of
    numbers whose largest, the product of a weight and a key's largest value A, is above
    2^10, so each is off by at most 2^-25, 2^-35 A over its key's own scale, and meets values
    below twice that scale: 2^-34 A for each key that is seen."""
    n, d = rows + 60, 64
    rng = np.random.default_rng(63)
    q, k, v = f32(rng, 1, 1, rows, d), f32(rng, 1, 1, n, d), f32(rng, 1, 1, n, d)
    v[0, 0, 30, 5] = 2.0 ** 18
    out = window(capi, q, k, v, workspace=workspace)
    check(out, q, k, v, [n], 0, 0, d ** -0.5)
    v[..., 5] = out[..., 5] = 0
    expected, bound = cases.attention(q, k, v, [n], None, 0, d ** -0.5)
    assert (np.abs(out - expected) <= bound + n * 2.0 ** -34 * 2.0 ** 18).all()


@pytest.mark.parametrize("workspace", [False, True])
def test_a_long_sum_of_small_weights(capi, workspace):
    """A weight of 1 and 32767 of just under half a step of it: a lane that added them one
    by one would lose its quarter of them, 8192 half steps, where the sums of
    sixteen lanes and more that the bound counts lose far less."""
    n, d = 32768, 16
    q, k, v = (np.zeros((1, 1, r, d), np.float32) for r in (16, n, n))
    q[..., 0], k[:, :, 0, 0], v[:, :, 0] = 1, 24.1, 1
    scale = float(np.float32(np.log(2)))
    out = window(capi, q, k, v, scale=scale, workspace=workspace)
    check(out, q, k, v, [n], 0, 0, scale)


def test_a_causal_prompt_of_thousands(capi):
    rng = np.random.default_rng(64)
    q, k, v = (f32(rng, 1, 1, 5000, 64) for _ in range(3))
    out = window(capi, np.ascontiguousarray(q[:, :, -16:]), k, v, workspace=False)
    check(out, q[:, :, -16:], k, v, [5000], 0, 0, 0.125)
    out = window(capi, np.ascontiguousarray(q[:, :, -1100:]), k, v)
    check(out[:, :, :20], q[:, :, -1100:-1080], k[:, :, :-1080], v[:, :, :-1080], [3920], 0, 0, 0.125)


@pytest.mark.parametrize("large", [1e4, 1e7, 1e12])
@pytest.mark.parametrize("shape,workspace", FORMS, ids=str)
def test_scores_without_fractions(capi, shape, workspace, large):
    """Scores so far apart that each row takes the value of one key alone, that of the
    largest product of small whole numbers: exact, where float32 scores have lost their
    fractions too, and however the maxima rise along the keys."""
    batch, heads, kv, rows, cols, d = shape
    rng = np.random.default_rng(66)
    q, k, v = np.zeros((batch, heads, rows, d), np.float32), np.zeros((batch, kv, cols, d), np.float32), f32(rng, batch, kv, cols, d)
    q[..., 0] = large
    k[..., 0] = np.arange(1, cols + 1) + 100 * (np.arange(cols) % 7 == 0)
    out = window(capi, q, k, v, scale=1.0, workspace=workspace)
    for b, h in form_heads(shape):
        best = np.maximum.accumulate(k[b, h // (heads // kv), :, 0])
        at = np.searchsorted(best, best[cols - rows:])  # the first key with it
        expected = v[b, h // (heads // kv), at]
        # The weight of one key alone is 1, its value held in halves.
        assert (np.abs(out[b, h] - expected) <= 2.0 ** -21 * np.abs(v[b, h // (heads // kv), at]).max(-1, keepdims=True)).all()


@pytest.mark.parametrize("heads,rows", [(1, 1), (4, 1), (2, 16)])
@pytest.mark.parametrize("features", [32, 64, 128])
@pytest.mark.parametrize("workspace", [False, True])
def test_small_cached_weights_beside_a_huge_value(capi, features, heads, rows, workspace):
    """The same in the 4-bit cache, of values that it holds exactly."""
    n = 8192
    q, k = np.zeros((1, heads, rows, features), np.float32), np.zeros((1, 1, n, features), np.float32)
    v = np.ones((1, 1, n, features), np.float32)
    q[..., :32] = 1 / 32
    k[:, :, 0, :32], v[:, :, 0] = 15, 2.0 ** 126
    scale = float(np.float32(np.log(2)))
    keys, values = cases.cache_rows(k), cases.cache_rows(v)
    np.testing.assert_array_equal(cases.cache_values(values, features), v)
    out = cached(capi, q, keys, values, [n], scale=scale, workspace=workspace)
    check(out, q, k, v, [n], 0, 0, scale)


@pytest.mark.parametrize("far", [(0, 2.0 ** 66), (0, 1e30), (2.0 ** -60, 2.0 ** 76), (0, 1e-20)], ids=str)
@pytest.mark.parametrize("heads,rows", [(4, 1), (2, 16)])
@pytest.mark.parametrize("features", [32, 64, 128])
def test_cached_values_far_apart(capi, features, heads, rows, far):
    rng = np.random.default_rng(65)
    n = 500
    q, k, v = f32(rng, 1, heads, rows, features), f32(rng, 1, 1, n, features), f32(rng, 1, 1, n, features)
    v[:, :, ::2] *= np.float32(far[0])
    v[:, :, 1::2] *= np.float32(far[1])
    keys, values = cases.cache_rows(k), cases.cache_rows(v)
    kk, vv = cases.cache_values(keys, features), cases.cache_values(values, features)
    for scale in (0.0, features ** -0.5):
        check(cached(capi, q, keys, values, [n], scale=scale), q, kk, vv, [n], 0, 0, scale)


@pytest.mark.parametrize("large", [1e4, 1e7, 1e12])
@pytest.mark.parametrize("heads,rows", [(1, 1), (4, 1), (2, 16)])
@pytest.mark.parametrize("features", [32, 64, 128])
def test_cached_scores_without_fractions(capi, features, heads, rows, large):
    """The same: tokens of whole numbers below 256, which the cache holds exactly."""
    n = 700
    rng = np.random.default_rng(67)
    q, k, v = np.zeros((1, heads, rows, features), np.float32), np.zeros((1, 1, n, features), np.float32), f32(rng, 1, 1, n, features)
    q[..., :32] = np.float32(large) / 32
    k[...] = (1 + np.arange(n) // 3 % 200 + 20 * (np.arange(n) % 7 == 0))[:, None]
    keys, values = cases.cache_rows(k), cases.cache_rows(v)
    np.testing.assert_array_equal(cases.cache_values(keys, features), k)
    out = cached(capi, q, keys, values, [n], scale=1.0)
    vv, best = cases.cache_values(values, features)[0, 0], k[0, 0, :, 0]
    for i in range(rows):
        seen = best[:n - rows + i + 1]
        expected = vv[:len(seen)][seen == seen.max()].mean(0)
        # Equal weights, products in halves, sums of a few.
        assert (np.abs(out[0, :, i] - expected) <= 2.0 ** -20 * np.abs(vv).max()).all()


# ------------------------------------------------------------------ beam selection
def select(capi, logits, scores, count):
    batch, beams, vocabulary = logits.shape
    dx, ds = capi.DeviceArray.from_numpy(logits), capi.DeviceArray.from_numpy(scores)
    outs = [capi.DeviceArray((batch, count)), *(capi.DeviceArray((batch, count), np.int32) for _ in range(2))]
    ws = capi.beam_select_workspace(batch, beams, vocabulary, count)
    capi.beam_select(dx.ptr, ds.ptr, *(o.ptr for o in outs), batch, beams, vocabulary, count, workspace=ws)
    capi.synchronize()
    return [o.numpy() for o in outs]


def check_selection(got, logits, scores, count):
    """The plain form's candidates, and their scores to half a step and 120 EPS of a
    float32 sum. Candidates of different beams whose scores are closer than such
    sums are may change places: the named ones' own scores have to be in order to that."""
    want, all_of = cases.beam_best(logits, scores, count), cases.beam_candidates(logits, scores)
    off = np.abs(got[0] - want[0])
    assert (off <= np.abs(want[0]) * EPS + 120 * EPS).all(), (off / EPS).max()
    named = all_of[np.arange(len(logits))[:, None], got[1], got[2]]
    assert (np.abs(named - want[0]) <= 120 * EPS).all()
    alone = np.diff(want[0], axis=-1, prepend=np.inf, append=-np.inf)
    alone = (np.abs(alone[:, :-1]) > 240 * EPS) & (np.abs(alone[:, 1:]) > 240 * EPS)
    alone[:, -1] = False  # what comes after it is not known
    np.testing.assert_array_equal(got[1][alone], want[1][alone])
    np.testing.assert_array_equal(got[2][alone], want[2][alone])
    chosen = got[1].astype(np.int64) * logits.shape[2] + got[2]
    assert all(len(np.unique(row)) == count for row in chosen)


@pytest.mark.parametrize("offset", [20.0, -200.0, 1000.0, -1e4, 1e5])
@pytest.mark.parametrize("shape", [(2, 3, 9000, 5), (16, 8, 40000, 4)], ids=str)
def test_select_of_logits_with_an_offset(capi, shape, offset):
    """A number added to a beam's logits, another for each beam, changes nothing: the
    sum of exponentials is one of differences from the maximum."""
    batch, beams, vocabulary, count = shape
    rng = np.random.default_rng(71)
    logits = 3 * f32(rng, batch, beams, vocabulary) + np.float32(offset) * (1 + f32(rng, batch, beams, 1) / 8)
    scores = f32(rng, batch, beams)
    check_selection(select(capi, logits, scores, count), logits, scores, count)


@pytest.mark.parametrize("top", [1000.0, -777.7, 12345.6])
def test_select_of_a_certain_token(capi, top):
    """One token far above the rest has a probability of 1, and its score is the beam's."""
    logits = np.full((1, 2, 20000), np.float32(top) - np.float32(1050), np.float32)
    logits[0, 0, 17] = logits[0, 1, 9000] = np.float32(top)
    got = select(capi, logits, np.array([[-1.5, -0.25]], np.float32), 2)
    np.testing.assert_array_equal(got[0], [[-0.25, -1.5]])
    assert got[1].tolist() == [[1, 0]] and got[2].tolist() == [[9000, 17]]


LOWEST = np.finfo(np.float32).min


@pytest.mark.parametrize("low", [LOWEST, np.float32(-3e38), np.float32(-2e38)], ids=str)
@pytest.mark.parametrize("shape", [(1, 4, 32000, 8), (16, 8, 40000, 16), (1, 2, 50, 3)], ids=str)
@pytest.mark.parametrize("kept", [0.01, 3])
def test_select_of_logits_masked_by_the_lowest_value(capi, shape, kept, low):
    """Tokens masked by float32's lowest value, in some parts of a row all of them: they
    weigh nothing beside others, and are candidates after those."""
    batch, beams, vocabulary, count = shape
    rng = np.random.default_rng(72)
    logits, scores = f32(rng, batch, beams, vocabulary), f32(rng, batch, beams)
    allowed = rng.random(logits.shape) < (kept if kept < 1 else 0)
    allowed[..., rng.permutation(vocabulary)[:3]] = True
    logits[~allowed] = low
    want, got = cases.beam_best(logits, scores, count), select(capi, logits, scores, count)
    real = want[0] > -1e30
    np.testing.assert_array_equal(got[1][real], want[1][real])
    np.testing.assert_array_equal(got[2][real], want[2][real])
    assert (np.abs(got[0] - want[0])[real] <= np.abs(want[0][real]) * EPS + 120 * EPS).all()
    with np.errstate(over="ignore"):
        np.testing.assert_allclose(got[0][~real], want[0][~real].astype(np.float32), rtol=2 * EPS)


@pytest.mark.parametrize("value", [LOWEST, np.float32(-2.5e38), np.float32(2.5e38), -LOWEST], ids=str)
@pytest.mark.parametrize("vocabulary", [100, 30000])
def test_select_of_equal_far_logits(capi, vocabulary, value):
    """All logits of a beam the same, near either end of float32: each has the probability
    of one in the vocabulary."""
    rng = np.random.default_rng(73)
    logits, scores = f32(rng, 1, 3, vocabulary) / 8, np.zeros((1, 3), np.float32)
    logits[0, 1] = value
    got = select(capi, logits, scores, 256)
    chosen = cases.beam_candidates(logits, scores)[0, got[1][0], got[2][0]]
    assert np.isfinite(got[0]).all()
    assert (np.abs(got[0][0] - chosen) <= np.abs(chosen) * EPS + 120 * EPS).all()


@pytest.mark.parametrize("shape", [(1, 8, 128256, 128), (1, 8, 32000, 256), (1, 64, 20000, 128), (3, 5, 9001, 200), (2, 64, 300, 256),
                                   (1, 16, 50000, 64)], ids=str)
def test_select_of_many_candidates(capi, shape):
    """Counts of which a merge has many thousand candidates."""
    batch, beams, vocabulary, count = shape
    rng = np.random.default_rng(74)
    logits, scores = 3 * f32(rng, batch, beams, vocabulary), f32(rng, batch, beams)
    check_selection(select(capi, logits, scores, count), logits, scores, count)


def test_select_behind_long_sequences(capi):
    """Scores of many tokens' logarithms: far from zero, and close together for their size."""
    rng = np.random.default_rng(75)
    logits, scores = 3 * f32(rng, 1, 16, 32000), (-800 + f32(rng, 1, 16)).astype(np.float32)
    for count in (16, 100, 256):
        check_selection(select(capi, logits, scores, count), logits, scores, count)


@pytest.mark.parametrize("beams,vocabulary,count", [(64, 300, 256), (8, 9001, 200), (3, 40000, 256)])
def test_select_of_ties_beside_finished_beams(capi, beams, vocabulary, count):
    """Candidates that all tie, of which a merge takes the heads of its lists one by one."""
    rng = np.random.default_rng(76)
    logits, scores = np.zeros((3, beams, vocabulary), np.float32), np.zeros((3, beams), np.float32)
    logits[1, :, ::3] = -np.inf
    scores[2, ::2] = -np.inf
    finished = rng.random((3, beams)) < 0.4
    finished[:, 0] = True
    dx, ds, df = (capi.DeviceArray.from_numpy(x) for x in (logits, scores, finished))
    outs = [capi.DeviceArray((3, count)), *(capi.DeviceArray((3, count), np.int32) for _ in range(2))]
    ws = capi.beam_select_workspace(3, beams, vocabulary, count)
    capi.beam_select(dx.ptr, ds.ptr, *(o.ptr for o in outs), 3, beams, vocabulary, count, finished=df.ptr, eos=7, workspace=ws)
    capi.synchronize()
    want = cases.beam_best(logits, scores, count, finished, 7)
    np.testing.assert_array_equal(outs[1].numpy(), want[1])
    np.testing.assert_array_equal(outs[2].numpy(), want[2])


def test_select_takes_alike_times_for_alike_counts(capi):
    """What the search leaves to be put in order depends on the count, not on what it has in
    common with the block's size: no count takes eight times as long as a larger one,
    where taking them one by one took seventy times and more."""
    rng = np.random.default_rng(77)
    batch, beams, vocabulary = 1, 8, 32000
    dx = capi.DeviceArray.from_numpy(3 * f32(rng, batch, beams, vocabulary))
    ds = capi.DeviceArray.from_numpy(f32(rng, batch, beams))
    outs = [capi.DeviceArray((batch, 256)), *(capi.DeviceArray((batch, 256), np.int32) for _ in range(2))]
    ws = capi.beam_select_workspace(batch, beams, vocabulary, 256)

    def seconds(count):
        taken = []
        for _ in range(5):
            capi.synchronize()
            start = time.perf_counter()
            for _ in range(4):
                capi.beam_select(dx.ptr, ds.ptr, *(o.ptr for o in outs), batch, beams, vocabulary, count, workspace=ws)
            capi.synchronize()
            taken.append(time.perf_counter() - start)
        return min(taken)
    times = {count: seconds(count) for count in (32, 64, 96, 128, 192, 256)}
    largest = seconds(250)
    assert all(taken < 8 * largest for taken in times.values()), (times, largest)
    assert largest < 20 * times[32], (times, largest)


@pytest.mark.parametrize("score", [-1e30, np.nan])
@pytest.mark.parametrize("count", [3, 200, 256])
def test_select_by_logits_alone(capi, count, score):
    """Scores that all round to the same, or are all NaN: the first beam's largest logits,
    found from thousands of candidates whose scores tie."""
    rng = np.random.default_rng(78)
    logits = f32(rng, 2, 8, 32000)
    got = select(capi, logits, np.full((2, 8), score, np.float32), count)
    for b in range(2):
        assert (got[1][b] == 0).all()
        np.testing.assert_array_equal(got[2][b], np.argsort(-logits[b, 0], kind="stable")[:count])
    np.testing.assert_array_equal(got[0], np.full((2, count), score, np.float32))
