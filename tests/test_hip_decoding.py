"""GPU tests of the decoding operators against plain 64-bit forms, through the C
ABI (strides, lengths, workspaces, streams, graphs) and through the package.

The tolerances are those that decoding_cases derives from float32's half step;
codes, tokens, beams and moved states are exact."""

from __future__ import annotations

import numpy as np
import pytest

import decoding_cases as cases
from conftest import require_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cx():
    require_gpu()
    import tensorcx
    return tensorcx


@pytest.fixture(scope="module")
def capi():
    require_gpu()
    import tensorcx_hip_capi
    return tensorcx_hip_capi


def hip(cx, a):
    return cx.tensor(a, device="hip")


def f32(rng, *shape):
    return rng.normal(size=shape).astype(np.float32)


def check_rows(out, expected, bound, context=""):
    assert out.shape == expected.shape and out.dtype == np.float32
    off = np.abs(out.astype(float) - expected)
    assert (off <= bound).all(), f"{context}: off by up to {np.nanmax(off / np.maximum(bound, 1e-300)):.3g} of the bound"


# (batch, heads, kv_heads, rows, cols, features, window, sinks, lengths)
SHAPES = [
    (1, 1, 1, 1, 1, 64, None, 0, None),            # one key
    (1, 1, 1, 1, 0, 64, None, 0, None),            # no key: zeros
    (2, 4, 2, 1, 100, 128, None, 0, [0, 100]),     # an empty sequence
    (3, 8, 2, 1, 333, 128, 17, 3, [333, 5, 64]),   # window and sinks of different lengths
    (2, 6, 6, 1, 70, 32, 1, 0, None),              # a window of the key itself
    (2, 6, 6, 1, 70, 32, 1, 70, None),             # sinks over everything
    (1, 5, 1, 1, 1025, 64, 200, 4, None),          # five heads on one
    (1, 16, 1, 1, 130, 64, None, 0, None),         # more heads than a block's rows
    (2, 3, 3, 7, 7, 64, None, 0, None),            # a prompt
    (1, 4, 2, 33, 65, 128, 16, 5, None),           # a chunk
    (2, 2, 1, 40, 31, 64, 8, 2, [31, 20]),         # more queries than keys: rows that see nothing
    (1, 4, 4, 200, 200, 64, 70, 65, None),         # sinks past a tile, a window across two
    (1, 2, 2, 129, 300, 32, 64, 64, None),
    (2, 8, 1, 65, 65, 128, 3, 0, [65, 64]),
    (1, 2, 1, 300, 1000, 64, 1000, 0, None),       # a window of all keys
    (1, 3, 1, 130, 700, 128, 90, 4, [650]),
    (1, 1, 1, 1, 20000, 64, None, 0, None),        # keys split over blocks
    (2, 4, 1, 3, 9000, 128, 5000, 7, [9000, 4097]),
]


def attention_inputs(rng, shape, features=None):
    batch, heads, kv, rows, cols, d, window, sinks, lengths = shape
    d = features or d
    q, k, v = f32(rng, batch, heads, rows, d), f32(rng, batch, kv, cols, d), f32(rng, batch, kv, cols, d)
    k += 2 * f32(rng, 1, kv, 1, d)
    return q, k, v, [cols] * batch if lengths is None else lengths


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_window_attention(cx, shape):
    rng = np.random.default_rng(11)
    q, k, v, lengths = attention_inputs(rng, shape)
    window, sinks = shape[6], shape[7]
    given = None if shape[8] is None else hip(cx, np.array(lengths, np.int32))
    expected, bound = cases.attention(q, k, v, lengths, window, sinks, shape[5] ** -0.5)
    out = cx.hip.window_attention(hip(cx, q), hip(cx, k), hip(cx, v), window, sinks, lengths=given)
    assert out.device == "hip" and out.dtype == "float32"
    check_rows(out.numpy(), expected, bound, str(shape))


@pytest.mark.parametrize("features", [16, 24, 40, 56, 72, 80, 96, 120])
@pytest.mark.parametrize("rows", [1, 50])
def test_window_attention_features(cx, features, rows):
    shape = (1, 4, 2, rows, 90, features, 30, 2, None)
    rng = np.random.default_rng(features)
    q, k, v, lengths = attention_inputs(rng, shape)
    expected, bound = cases.attention(q, k, v, lengths, 30, 2, 0.3)
    out = cx.hip.window_attention(hip(cx, q), hip(cx, k), hip(cx, v), 30, 2, scale=0.3)
    check_rows(out.numpy(), expected, bound)


@pytest.mark.parametrize("scale", [0.0, -0.25, 3.0])
@pytest.mark.parametrize("rows", [1, 70])
def test_window_attention_scales(cx, scale, rows):
    rng = np.random.default_rng(5)
    q, k, v, lengths = attention_inputs(rng, (1, 2, 2, rows, 130, 64, 100, 3, None))
    expected, bound = cases.attention(q, k, v, lengths, 100, 3, scale)
    check_rows(cx.hip.window_attention(hip(cx, q), hip(cx, k), hip(cx, v), 100, 3, scale=scale).numpy(), expected, bound)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("rows", [1, 2, 150])
def test_hidden_keys_have_no_influence(cx, bad, rows):
    """Keys behind a sequence's end, before its window and after its queries hold
    anything: no output changes by a bit."""
    rng = np.random.default_rng(8)
    shape = (2, 4, 2, rows, 400, 64, 60, 3, [330, 300])
    q, k, v, lengths = attention_inputs(rng, shape)
    n = hip(cx, np.array(lengths, np.int32))
    clean = cx.hip.window_attention(hip(cx, q), hip(cx, k), hip(cx, v), 60, 3, lengths=n).numpy()
    for b, length in enumerate(lengths):
        k[b, :, length:], v[b, :, length:] = bad, bad
        first = length - rows - 60 + 1  # the window of the first query
        if first > 3:
            k[b, :, 3:first], v[b, :, 3:first] = bad, bad
    again = cx.hip.window_attention(hip(cx, q), hip(cx, k), hip(cx, v), 60, 3, lengths=n).numpy()
    np.testing.assert_array_equal(again.view(np.uint32), clean.view(np.uint32))


@pytest.mark.parametrize("rows", [1, 4, 150])
def test_a_bad_key_reaches_only_the_rows_that_see_it(cx, rows):
    """NaN in one key or value: the rows that see it are NaN (of a value, in its
    feature), the others stay as they are to their bounds."""
    rng = np.random.default_rng(9)
    q, k, v, lengths = attention_inputs(rng, (1, 4, 2, rows, 200, 64, 40, 2, None))
    expected, bound = cases.attention(q, k, v, lengths, 40, 2, 0.125)
    for where in (195, 170, 0):
        seen = cases.visible(rows, 200, 200, 40, 2)[:, where]
        kk, vv = k.copy(), v.copy()
        kk[0, 0, where, 5] = np.nan
        out = cx.hip.window_attention(hip(cx, q), hip(cx, kk), hip(cx, v), 40, 2).numpy()
        assert np.isnan(out[0, :2][:, seen]).all()
        fine = np.ones(out.shape, bool)
        fine[0, :2] &= ~seen[None, :, None]
        assert (np.abs(out - expected)[fine] <= np.broadcast_to(bound, out.shape)[fine]).all()
        vv[0, 1, where, 7] = np.nan
        out = cx.hip.window_attention(hip(cx, q), hip(cx, k), hip(cx, vv), 40, 2).numpy()
        fine = np.ones(out.shape, bool)
        fine[0, 2:, :, 7] &= ~seen[None]
        assert np.isnan(out[~fine]).all()
        assert (np.abs(out - expected)[fine] <= np.broadcast_to(bound, out.shape)[fine]).all()


@pytest.mark.parametrize("rows", [1, 100])
def test_far_scales_of_heads_and_features(cx, rows):
    """Values of one feature 10^4 times the others', keys of one token 10^3 times
    the others', tiny and huge tensors: errors stay relative to their own feature
    (values) and score (keys)."""
    rng = np.random.default_rng(10)
    q, k, v, lengths = attention_inputs(rng, (1, 2, 1, rows, 300, 64, 200, 4, None))
    v[..., 3] *= 1e4
    out = cx.hip.window_attention(hip(cx, q), hip(cx, k), hip(cx, v), 200, 4).numpy()
    small = np.delete(v, 3, -1)
    expected, bound = cases.attention(q, k, v, lengths, 200, 4, 0.125)
    keep = [f for f in range(64) if f != 3]
    ratio = np.abs(small).max() / np.abs(v).max()
    assert (np.abs(out - expected)[..., keep] <= (bound * ratio * 1.01)[..., :]).all()
    v2 = (f32(rng, 1, 1, 300, 64) * np.float32(1e30)).astype(np.float32)
    expected, bound = cases.attention(q, k, v2, lengths, 200, 4, 0.125)
    check_rows(cx.hip.window_attention(hip(cx, q), hip(cx, k), hip(cx, v2), 200, 4).numpy(), expected, bound)
    k2, q2 = (k * np.float32(1e-20)).astype(np.float32), (q * np.float32(1e20)).astype(np.float32)
    expected, bound = cases.attention(q2, k2, v, lengths, 200, 4, 0.125)
    check_rows(cx.hip.window_attention(hip(cx, q2), hip(cx, k2), hip(cx, v), 200, 4).numpy(), expected, bound)


@pytest.mark.parametrize("rows", [1, 90])
def test_strides_and_workspaces(capi, rows):
    """Token-major tensors with gaps, lengths on the device, every workspace from
    none to all: results inside the bound, and nothing written between rows."""
    rng = np.random.default_rng(12)
    batch, heads, kv, cols, d = 2, 4, 2, 3000, 64
    q, k, v, lengths = attention_inputs(rng, (batch, heads, kv, rows, cols, d, None, 0, [2900, 1500]))
    expected, bound = cases.attention(q, k, v, lengths, 2000, 5, 0.125)

    def token_major(x, gap):
        y = np.full((x.shape[0], x.shape[2], x.shape[1], x.shape[3] + gap), np.float32(7))
        y[..., :x.shape[3]] = x.transpose(0, 2, 1, 3)
        return y

    def strides(y):
        return [y.strides[0] // 4, y.strides[2] // 4, y.strides[1] // 4]
    qt, kt, vt, ot = token_major(q, 4), token_major(k, 8), token_major(v, 0), token_major(np.zeros_like(q), 12)
    dq, dk, dv, dn = (capi.DeviceArray.from_numpy(x) for x in (qt, kt, vt, np.array(lengths, np.int32)))
    desc = capi.window_attention_desc(batch, heads, kv, rows, cols, d, window=2000, sinks=5, lengths=dn.ptr,
                                      q_strides=strides(qt), k_strides=strides(kt), v_strides=strides(vt),
                                      out_strides=strides(ot))
    whole = capi.window_attention_workspace(desc)
    for part in (0.0, 0.3, 1.0):
        out = capi.DeviceArray.from_numpy(ot)
        ws = capi.Workspace(whole.address, int(whole.nbytes * part)) if whole is not None and part else None
        capi.window_attention(dq.ptr, dk.ptr, dv.ptr, out.ptr, desc, workspace=ws)
        capi.synchronize()
        got = out.numpy()
        check_rows(np.ascontiguousarray(got[..., :d].transpose(0, 2, 1, 3)), expected, bound, f"part {part}")
        np.testing.assert_array_equal(got[..., d:], ot[..., d:])


def test_lengths_out_of_range(cx, capi):
    rng = np.random.default_rng(13)
    q, k, v, _ = attention_inputs(rng, (3, 2, 2, 1, 50, 64, None, 0, None))
    lengths = np.array([-5, 51, 20], np.int32)
    with pytest.raises(ValueError, match="lengths"):
        cx.hip.window_attention(hip(cx, q), hip(cx, k), hip(cx, v), lengths=hip(cx, lengths))
    arrays = [capi.DeviceArray.from_numpy(x) for x in (q, k, v, np.zeros_like(q), lengths)]
    desc = capi.window_attention_desc(3, 2, 2, 1, 50, 64, lengths=arrays[4].ptr)
    capi.window_attention(*(a.ptr for a in arrays[:4]), desc)
    capi.synchronize()
    expected, bound = cases.attention(q, k, v, [0, 50, 20], None, 0, 0.125)
    check_rows(arrays[3].numpy(), expected, bound)


# ------------------------------------------------------------------ the 4-bit cache
def special_tokens(rng, features):
    """Tokens whose groups are constant, tiny, huge, of one sign, far from zero,
    subnormal, non-finite, or tie between two codes."""
    x = f32(rng, 1, 2, 24, features)
    x[0, 0, 0] = 0
    x[0, 0, 1] = -0.0
    x[0, 0, 2] = 3.25
    x[0, 0, 3] = -7.1
    x[0, 0, 4] *= 1e-38
    x[0, 0, 5] *= 1e-44
    x[0, 0, 6] *= 1e37
    x[0, 0, 7] = np.where(x[0, 0, 7] > 0, np.float32(3.4e38), np.float32(-3.4e38))
    x[0, 0, 8, 3] = np.nan
    x[0, 0, 9, features - 1] = np.inf
    x[0, 0, 10, 16] = -np.inf
    x[0, 0, 11] = 1000 + x[0, 0, 11]
    x[0, 0, 12] = -1000 + x[0, 0, 12] * np.float32(1e-3)
    x[0, 0, 13] = np.arange(features) % 32 * np.float32(0.5)  # ties
    x[0, 0, 14] = -np.abs(x[0, 0, 14])
    x[0, 0, 15] = np.arange(features, dtype=np.float32) / 7
    return x


@pytest.mark.parametrize("features", [32, 64, 128])
def test_store_and_load(cx, features):
    rng = np.random.default_rng(features)
    x = special_tokens(rng, features)
    y = f32(rng, *x.shape)
    keys, values = cx.hip.new_cache(1, 2, 40, features), cx.hip.new_cache(1, 2, 40, features)
    assert keys.shape == (1, 2, 40, features // 8 + features // 32) and keys.dtype == "int32"
    before = rng.integers(-2 ** 31, 2 ** 31 - 1, keys.shape).astype(np.int32)
    keys = hip(cx, before)
    cx.hip.cache_store(hip(cx, x), hip(cx, y), keys, values, hip(cx, np.array([9], np.int32)))
    got = keys.numpy()
    np.testing.assert_array_equal(got[:, :, 9:33], cases.cache_rows(x))
    np.testing.assert_array_equal(values.numpy()[:, :, 9:33], cases.cache_rows(y))
    # Slots before and after stay as they were.
    np.testing.assert_array_equal(got[:, :, :9], before[:, :, :9])
    np.testing.assert_array_equal(got[:, :, 33:], before[:, :, 33:])
    read = cx.hip.cache_load(keys, 9, 24)
    assert read.shape == x.shape and read.dtype == "float32"
    expected = cases.cache_values(got[:, :, 9:33], features)
    # One rounding of low + step * code, or none.
    np.testing.assert_allclose(read.numpy(), expected, rtol=cases.EPS, atol=2.0 ** -150, equal_nan=True)
    assert cx.hip.cache_load(keys, 40).shape == (1, 2, 0, features)
    assert cx.hip.cache_load(values).shape == (1, 2, 40, features)
    with pytest.raises(ValueError):
        cx.hip.cache_load(keys, 30, 11)


@pytest.mark.parametrize("features", [32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 5, 70])
def test_store_of_ragged_batches(capi, features, tokens):
    """Token-major keys and values, a position for each sequence; tokens past the
    capacity are dropped and flagged, tokens in range are stored all the same."""
    rng = np.random.default_rng(4)
    batch, kv, capacity = 5, 3, 90
    x, y = f32(rng, batch, tokens, kv, features + 4), f32(rng, batch, tokens, kv, features)
    positions = np.array([0, 7, capacity - tokens, capacity - tokens + 1, -1], np.int32)
    words = capi.cache4_words(features)
    before = rng.integers(-2 ** 31, 2 ** 31 - 1, (batch, kv, capacity, words)).astype(np.int32)
    dx, dy, dp, keys, values = (capi.DeviceArray.from_numpy(a) for a in (x, y, positions, before, before))
    import ctypes
    flag = ctypes.c_void_p()
    capi.check(capi.lib().tcx_hip_flag_acquire(ctypes.byref(flag)))
    desc = capi.cache4_store_desc(batch, kv, tokens, capacity, features, flag=flag.value,
                                  key_strides=(tokens * kv * (features + 4), features + 4, kv * (features + 4)),
                                  value_strides=(tokens * kv * features, features, kv * features))
    capi.cache4_store(dx.ptr, dy.ptr, keys.ptr, values.ptr, dp.ptr, desc)
    capi.synchronize()
    assert ctypes.c_int32.from_address(flag.value).value == 1
    capi.lib().tcx_hip_flag_release(flag)
    for source, cache in ((x[..., :features], keys), (y, values)):
        expected = before.copy()
        rows = cases.cache_rows(np.ascontiguousarray(source.transpose(0, 2, 1, 3)))
        for b, p in enumerate(positions):
            for t in range(tokens):
                if 0 <= p + t < capacity:
                    expected[b, :, p + t] = rows[b, :, t]
        np.testing.assert_array_equal(cache.numpy(), expected)


@pytest.mark.parametrize("features", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_cache_attention(cx, shape, features):
    rng = np.random.default_rng(21)
    q, k, v, lengths = attention_inputs(rng, shape, features)
    keys, values = cases.cache_rows(k), cases.cache_rows(v)
    window, sinks = shape[6], shape[7]
    expected, bound = cases.attention(q, cases.cache_values(keys, features), cases.cache_values(values, features), lengths,
                                      window, sinks, features ** -0.5)
    out = cx.hip.cache_attention(hip(cx, q), hip(cx, keys), hip(cx, values), hip(cx, np.array(lengths, np.int32)), window,
                                 sinks)
    check_rows(out.numpy(), expected, bound, str(shape))


@pytest.mark.parametrize("rows", [1, 20])
def test_cache_attention_hides_what_is_behind(cx, rows):
    """Slots outside a sequence's keys hold any words, NaN scales among them."""
    rng = np.random.default_rng(22)
    q, k, v, lengths = attention_inputs(rng, (2, 8, 2, rows, 500, 128, 70, 3, [480, 300]))
    keys, values = cases.cache_rows(k), cases.cache_rows(v)
    n = hip(cx, np.array(lengths, np.int32))
    clean = cx.hip.cache_attention(hip(cx, q), hip(cx, keys), hip(cx, values), n, 70, 3).numpy()
    for b, length in enumerate(lengths):
        for part in (np.s_[length:], np.s_[3:length - rows - 70 + 1]):
            keys[b, :, part] = rng.integers(-2 ** 31, 2 ** 31 - 1, keys[b, :, part].shape)
            values[b, :, part] = 0x7fc07fc0
    again = cx.hip.cache_attention(hip(cx, q), hip(cx, keys), hip(cx, values), n, 70, 3).numpy()
    np.testing.assert_array_equal(again.view(np.uint32), clean.view(np.uint32))


def test_cache_attention_of_far_scales(cx):
    """Groups of values whose steps differ by 10^5, tokens of tiny and huge values."""
    rng = np.random.default_rng(23)
    q, k, v, lengths = attention_inputs(rng, (1, 4, 1, 1, 700, 128, None, 0, None))
    v[..., 32:64] *= 1e-5
    v[:, :, ::7] *= 1e3
    k[:, :, ::5] *= 1e-3
    keys, values = cases.cache_rows(k), cases.cache_rows(v)
    vv = cases.cache_values(values, 128)
    expected, bound = cases.attention(q, cases.cache_values(keys, 128), vv, lengths, None, 0, 128 ** -0.5)
    out = cx.hip.cache_attention(hip(cx, q), hip(cx, keys), hip(cx, values), hip(cx, np.array(lengths, np.int32))).numpy()
    check_rows(out, expected, bound)
    group = np.abs(vv[..., 32:64]).max() / np.abs(vv).max()
    assert (np.abs(out - expected)[..., 32:64] <= bound * group * 1.01).all()


@pytest.mark.parametrize("heads,rows", [(2, 1), (8, 1), (2, 16)])
@pytest.mark.parametrize("features", [32, 64, 128])
def test_cache_attention_of_many_alike(cx, features, heads, rows):
    """Outputs that are means of many values are exact to their own size.

    Such sums cancel as the exact ones do: a term's error is a weight's (two halves of 22
    bits, exp2 and the score, some 2^-22 together) times a value, so the root mean
    square over the outputs is some 2^-21 of theirs; eight times that is allowed."""
    rng = np.random.default_rng(25)
    q, k, v = f32(rng, 1, heads, rows, features), f32(rng, 1, 2, 512, features), f32(rng, 1, 2, 512, features)
    keys, values = cases.cache_rows(k), cases.cache_rows(v)
    expected, _ = cases.attention(q, cases.cache_values(keys, features), cases.cache_values(values, features), [512], None,
                                  0, features ** -0.5)
    out = cx.hip.cache_attention(hip(cx, q), hip(cx, keys), hip(cx, values), hip(cx, np.array([512], np.int32))).numpy()
    assert np.sqrt(((out - expected) ** 2).mean()) <= 2.0 ** -18 * np.sqrt((expected ** 2).mean())


def test_a_lost_group_makes_its_readers_nan(cx):
    rng = np.random.default_rng(24)
    q, k, v, lengths = attention_inputs(rng, (1, 4, 2, 1, 100, 64, None, 0, None))
    k[0, 0, 50, 3] = np.inf
    v[0, 1, 60, 40] = np.nan
    n = hip(cx, np.array(lengths, np.int32))
    out = cx.hip.cache_attention(hip(cx, q), hip(cx, cases.cache_rows(k)), hip(cx, cases.cache_rows(v)), n).numpy()
    assert np.isnan(out[0, :2]).all() and np.isnan(out[0, 2:, :, 32:]).all() and np.isfinite(out[0, 2:, :, :32]).all()


# ------------------------------------------------------------------ beam search
@pytest.mark.parametrize("batch,beams,vocabulary,count", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 21), (1, 4, 300, 8), (3, 2, 8192, 4), (2, 5, 8193, 10), (1, 4, 32000, 8),
    (2, 8, 50257, 16), (1, 2, 128256, 4), (1, 64, 1000, 128), (1, 3, 20000, 256), (4, 1, 100, 100)])
def test_beam_select(cx, batch, beams, vocabulary, count):
    rng = np.random.default_rng(vocabulary + count)
    logits, scores = 3 * f32(rng, batch, beams, vocabulary), f32(rng, batch, beams) - 5
    expected = cases.beam_best(logits, scores, count)
    got = cx.hip.beam_select(hip(cx, logits), hip(cx, scores), count)
    np.testing.assert_array_equal(got[1].numpy(), expected[1])
    np.testing.assert_array_equal(got[2].numpy(), expected[2])
    # The maximum and the score are exact; the sum of exponentials is good to a
    # few EPS of each term and of the sums of 32, 64 and 4 terms, and the result
    # is rounded once.
    limit = np.abs(expected[0]) * cases.EPS + 120 * cases.EPS
    assert (np.abs(got[0].numpy() - expected[0]) <= limit).all()


def test_beam_select_ties(cx):
    """Equal logits over parts of the vocabulary, equal beams, -0 and +0: the lower
    token, then the lower beam."""
    logits = np.zeros((1, 3, 20000), np.float32)
    logits[0, 1, ::2] = -0.0
    scores = np.zeros((1, 3), np.float32)
    for count in (1, 7, 200):
        _, beams, tokens = cx.hip.beam_select(hip(cx, logits), hip(cx, scores), count)
        np.testing.assert_array_equal(beams.numpy()[0], np.zeros(count, np.int32))
        np.testing.assert_array_equal(tokens.numpy()[0], np.arange(count))
    logits[0, :, 15000] = 4
    logits[0, :, 9000] = 4
    _, beams, tokens = cx.hip.beam_select(hip(cx, logits), hip(cx, scores), 6)
    assert beams.numpy()[0].tolist() == [0, 0, 1, 1, 2, 2] and tokens.numpy()[0].tolist() == [9000, 15000] * 3


def test_beam_select_finished(cx):
    rng = np.random.default_rng(31)
    logits, scores = 2 * f32(rng, 3, 4, 500), f32(rng, 3, 4) - 3
    finished = np.array([[1, 0, 0, 1], [0, 0, 0, 0], [1, 1, 1, 1]], bool)
    for count in (4, 12):
        expected = cases.beam_best(logits, scores, count, finished, 7)
        got = cx.hip.beam_select(hip(cx, logits), hip(cx, scores), count, finished=hip(cx, finished), eos=7)
        np.testing.assert_array_equal(got[1].numpy(), expected[1])
        np.testing.assert_array_equal(got[2].numpy(), expected[2])
        with np.errstate(all="ignore"):
            off = np.where(np.isneginf(expected[0]), 0, np.abs(got[0].numpy() - expected[0]))
        assert (off <= np.abs(np.where(np.isneginf(expected[0]), 0, expected[0])) * cases.EPS + 120 * cases.EPS).all()
        assert (np.isneginf(got[0].numpy()) == np.isneginf(expected[0])).all()


def test_beam_select_dead_beams_and_banned_tokens(cx):
    """-inf logits and scores come last, by index; a beam of nothing but -inf offers -inf."""
    rng = np.random.default_rng(32)
    logits, scores = f32(rng, 2, 3, 40), f32(rng, 2, 3)
    logits[0, 0] = -np.inf
    logits[0, 1, 3:] = -np.inf
    scores[0, 2] = -np.inf
    logits[1, :, 1:] = -np.inf
    expected = cases.beam_best(logits, scores, 10)
    got = cx.hip.beam_select(hip(cx, logits), hip(cx, scores), 10)
    np.testing.assert_array_equal(got[1].numpy(), expected[1])
    np.testing.assert_array_equal(got[2].numpy(), expected[2])
    assert (np.isneginf(got[0].numpy()) == np.isneginf(expected[0])).all() and not np.isnan(got[0].numpy()).any()


def test_beam_select_nan(cx):
    rng = np.random.default_rng(33)
    logits, scores = f32(rng, 1, 3, 100), np.zeros((1, 3), np.float32)
    logits[0, 1, 17] = np.nan
    values, beams, tokens = cx.hip.beam_select(hip(cx, logits), hip(cx, scores), 2)
    assert np.isnan(values.numpy()).all() and beams.numpy().tolist() == [[1, 1]] and tokens.numpy()[0, 0] == 17


def test_beam_select_refusals(cx):
    x, s = hip(cx, np.zeros((1, 2, 10), np.float32)), hip(cx, np.zeros((1, 2), np.float32))
    done = hip(cx, np.zeros((1, 2), bool))
    for call in (lambda: cx.hip.beam_select(x, s, 21), lambda: cx.hip.beam_select(x, s, 0),
                 lambda: cx.hip.beam_select(x, s, 2, finished=done, eos=10), lambda: cx.hip.beam_select(x, x, 2),
                 lambda: cx.hip.beam_select(x, s, 2, finished=s, eos=1), lambda: cx.hip.beam_select(s, s, 2),
                 lambda: cx.hip.beam_select(hip(cx, np.zeros((1, 2, 10), np.int32)), s, 2)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("width", [1, 3, 4, 31, 1000, 4096, 70001])
def test_beam_reorder(cx, width):
    rng = np.random.default_rng(width)
    batch, beams, count = 3, 4, 5
    a = f32(rng, batch * beams, width)
    b = rng.integers(-2 ** 31, 2 ** 31 - 1, (batch * beams, 2, width)).astype(np.int32)
    c = rng.random((batch * beams, width)) < 0.5
    states = [hip(cx, x) for x in (a, b, c)] * 4  # more tensors than one launch takes
    index = rng.integers(0, beams, (batch, count)).astype(np.int32)
    rows = (np.arange(batch)[:, None] * beams + index).reshape(-1)
    out = cx.hip.beam_reorder(states, hip(cx, index))
    for got, x in zip(out, [a, b, c] * 4):
        assert got.shape == (batch * count, *x.shape[1:])
        np.testing.assert_array_equal(got.numpy(), x[rows])
    single = cx.hip.beam_reorder(states[0], hip(cx, index))
    np.testing.assert_array_equal(single.numpy(), a[rows])


def test_beam_reorder_refuses(cx):
    a = hip(cx, np.zeros((6, 8), np.float32))
    index = np.array([[0, 2], [1, 3]], np.int32)
    with pytest.raises(ValueError, match="beam"):
        cx.hip.beam_reorder(a, hip(cx, index))
    for bad in (np.zeros((4, 1), np.int32), np.zeros((2, 2), np.float32), np.zeros(2, np.int32)):
        with pytest.raises(ValueError):
            cx.hip.beam_reorder(a, hip(cx, bad))
    assert cx.hip.beam_reorder(hip(cx, np.zeros((6, 0), np.float32)), hip(cx, np.zeros((2, 1), np.int32))).shape == (2, 0)


def test_attention_refusals(cx):
    def z(*shape, dtype=np.float32):
        return hip(cx, np.zeros(shape, dtype))
    q, k, n = z(2, 4, 1, 64), z(2, 2, 8, 64), z(2, dtype=np.int32)
    cache = cx.hip.new_cache(2, 2, 8, 64)
    w, c = cx.hip.window_attention, cx.hip.cache_attention
    for call in (lambda: w(q, k, z(2, 2, 7, 64)), lambda: w(q, z(1, 2, 8, 64), z(1, 2, 8, 64)), lambda: w(q, z(2, 3, 8, 64), z(2, 3, 8, 64)),
                 lambda: w(q, z(2, 2, 8, 32), z(2, 2, 8, 32)), lambda: w(z(2, 4, 1, 20), z(2, 2, 8, 20), z(2, 2, 8, 20)),
                 lambda: w(q, k, k, 0), lambda: w(q, k, k, -3), lambda: w(q, k, k, 1, -1), lambda: w(z(2, 4, 64), k, k),
                 lambda: w(q, k, k, lengths=z(3, dtype=np.int32)), lambda: w(q, k, k, lengths=z(2)),
                 lambda: w(q, cache, cache), lambda: w(q, k, k, scale=float("nan")), lambda: w(q, k, k, scale=1e300),
                 lambda: c(q, cache, cx.hip.new_cache(2, 2, 9, 64), n), lambda: c(q, k, k, n),
                 lambda: c(z(2, 4, 1, 128), cache, cache, n), lambda: c(q, cache, cache, z(2)),
                 lambda: cx.hip.cache_store(k, k, cache, cache, n),  # one cache for both
                 lambda: cx.hip.cache_store(k, k, cache, cx.hip.new_cache(2, 2, 9, 64), n),
                 lambda: cx.hip.cache_store(k, z(2, 2, 7, 64), cache, cx.hip.new_cache(2, 2, 8, 64), n),
                 lambda: cx.hip.cache_store(k, k, cache, cx.hip.new_cache(2, 2, 8, 64), z(2))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: w(q, k, k, True), lambda: w(q, k, k, 1.5), lambda: w(q, k, k, 1, "2"), lambda: w(q, k, k, scale="1")):
        with pytest.raises(TypeError):
            call()
    assert w(z(0, 4, 1, 64), z(0, 2, 8, 64), z(0, 2, 8, 64)).shape == (0, 4, 1, 64)


# ------------------------------------------------------------------ together
def test_a_decoding_loop(cx):
    """Beam search over a small model: prompt by window attention, the keys and
    values stored in 4 bits, then steps of store, attention, selection and
    reordering. Every step's operators are checked against the plain forms on the
    states that the device holds."""
    rng = np.random.default_rng(77)
    batch, beams, heads, kv, d, vocabulary, capacity, window, sinks = 2, 3, 4, 2, 64, 400, 64, 24, 2
    prompt = 20
    width = heads * d
    make = lambda *s: hip(cx, (f32(rng, *s) * s[-1] ** -0.5).astype(np.float32))
    table, wq, wk, wv, head = make(vocabulary, width), make(heads * d, width), make(kv * d, width), make(kv * d, width), make(vocabulary, width)

    def project(x, w, n_heads, rows, tokens):
        return cx.transpose(cx.linear(x, w).reshape((rows, tokens, n_heads, d)), (0, 2, 1, 3))

    ids = rng.integers(0, vocabulary, (batch, prompt)).astype(np.int32)
    x = cx.embedding(hip(cx, ids), table)
    q, k, v = project(x, wq, heads, batch, prompt), project(x, wk, kv, batch, prompt), project(x, wv, kv, batch, prompt)
    mixed = cx.hip.window_attention(q, k, v, window, sinks)
    expected, bound = cases.attention(q.numpy(), k.numpy(), v.numpy(), [prompt] * batch, window, sinks, d ** -0.5)
    check_rows(mixed.numpy(), expected, bound, "prompt")
    keys, values = cx.hip.new_cache(batch, kv, capacity, d), cx.hip.new_cache(batch, kv, capacity, d)
    cx.hip.cache_store(k, v, keys, values, cx.zeros((batch,), "int32", "hip"))
    # Every beam starts as its sequence's prompt, and only the first counts.
    spread = hip(cx, np.zeros((batch, beams), np.int32))
    keys, values = cx.hip.beam_reorder([keys, values], spread)
    logits = cx.linear(cx.transpose(mixed, (0, 2, 1, 3)).reshape((batch, prompt, width))[:, -1], head)
    logits = hip(cx, np.repeat(logits.numpy()[:, None], beams, 1))
    scores = np.full((batch, beams), -np.inf, np.float32)
    scores[:, 0] = 0
    scores, finished = hip(cx, scores), np.zeros((batch, beams), bool)
    rows = batch * beams
    for step in range(12):
        want = cases.beam_best(logits.numpy(), scores.numpy(), beams, finished, 1)
        scores, parents, tokens = cx.hip.beam_select(logits, scores, beams, finished=hip(cx, finished), eos=1)
        np.testing.assert_array_equal(parents.numpy(), want[1])
        np.testing.assert_array_equal(tokens.numpy(), want[2])
        source = (np.arange(batch)[:, None] * beams + want[1]).reshape(-1)
        old = keys.numpy(), values.numpy()
        keys, values = cx.hip.beam_reorder([keys, values], parents)
        np.testing.assert_array_equal(keys.numpy(), old[0][source])
        np.testing.assert_array_equal(values.numpy(), old[1][source])
        finished = np.take_along_axis(finished, want[1], 1) | (want[2] == 1)
        x = cx.embedding(tokens.reshape((rows, 1)), table)
        q, k, v = project(x, wq, heads, rows, 1), project(x, wk, kv, rows, 1), project(x, wv, kv, rows, 1)
        at = np.full(rows, prompt + step, np.int32)
        cx.hip.cache_store(k, v, keys, values, hip(cx, at))
        np.testing.assert_array_equal(keys.numpy()[:, :, prompt + step], cases.cache_rows(k.numpy())[:, :, 0])
        mixed = cx.hip.cache_attention(q, keys, values, hip(cx, at + 1), window, sinks)
        expected, bound = cases.attention(q.numpy(), cases.cache_values(keys.numpy(), d), cases.cache_values(values.numpy(), d),
                                          at + 1, window, sinks, d ** -0.5)
        check_rows(mixed.numpy(), expected, bound, f"step {step}")
        logits = cx.linear(mixed.reshape((rows, width)), head).reshape((batch, beams, vocabulary))
