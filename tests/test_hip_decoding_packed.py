"""GPU tests of windowed attention from packed tiles, which large prompts take when
they have the workspace that they ask for: what hides in a tile that some rows share, values that
are not finite, empty sequences, strides; and of the cache attention's strides,
workspaces and lengths.

Tolerances are those of decoding_cases; what must not change is compared bit by bit."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import decoding_cases as cases
from conftest import require_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    require_gpu()
    import tensorcx_hip_capi
    assert tensorcx_hip_capi.available()
    return tensorcx_hip_capi


def f32(rng, *shape):
    return rng.normal(size=shape).astype(np.float32)


# (batch, heads, kv_heads, rows, cols, features, window, sinks): blocks of 64 rows, of 128
# and of 256.
PACKED = [
    (1, 1, 1, 1030, 1100, 64, 100, 3),
    (1, 2, 1, 600, 700, 128, 90, 70),
    (43, 2, 2, 257, 300, 32, 70, 5),
    (43, 2, 2, 257, 270, 128, 0, 0),
    (128, 1, 1, 300, 320, 80, 70, 2),
]


def packed_bytes(shape):
    batch, _, kv, _, cols, features = shape[:6]
    return batch * kv * cols * (32 if features <= 32 else 64 if features <= 64 else 128) * 8


def strides(y):
    """Of a (batch, tokens, heads, features) array, as (sequence, head, token)."""
    return [y.strides[0] // 4, y.strides[2] // 4, y.strides[1] // 4]


def run(capi, shape, q, k, v, lengths=None, **more):
    batch, heads, kv, rows, cols, d, window, sinks = shape
    dq, dk, dv = (capi.DeviceArray.from_numpy(x) for x in (q, k, v))
    out = capi.DeviceArray.from_numpy(np.full((batch, heads, rows, d), 7, np.float32))
    dn = None if lengths is None else capi.DeviceArray.from_numpy(np.asarray(lengths, np.int32))
    desc = capi.window_attention_desc(batch, heads, kv, rows, cols, d, window=window, sinks=sinks,
                                      lengths=None if dn is None else dn.ptr, **more)
    ws = capi.window_attention_workspace(desc)
    assert ws is not None and ws.nbytes >= packed_bytes(shape) * 0.2  # of a window's tiles alone
    capi.window_attention(dq.ptr, dk.ptr, dv.ptr, out.ptr, desc, workspace=ws)
    capi.synchronize()
    return out.numpy()


def inputs(shape, seed):
    batch, heads, kv, rows, cols, d = shape[:6]
    rng = np.random.default_rng(seed)
    return f32(rng, batch, heads, rows, d), f32(rng, batch, kv, cols, d), f32(rng, batch, kv, cols, d)


def some_heads(shape):
    return sorted({(0, 0), (shape[0] // 2, shape[1] - 1), (shape[0] - 1, 0)})


def plain(shape, q, k, v, lengths, b, h):
    share = shape[1] // shape[2]
    key = np.s_[b:b + 1, h // share:h // share + 1]
    expected, bound = cases.attention(q[b:b + 1, h:h + 1], k[key], v[key], lengths[b:b + 1], shape[6] or None, shape[7],
                                      shape[5] ** -0.5)
    return expected[0, 0], bound[0, 0]


def lengths_of(shape):
    batch, _, _, rows, cols = shape[:5]
    n = np.random.default_rng(batch).integers(rows // 2, cols + 1, batch)
    n[0] = cols - 13
    return n


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("shape", PACKED, ids=str)
def test_hidden_keys_have_no_influence(capi, shape, bad):
    """Keys behind a sequence's end and before its first query's window hold anything, in
    tiles whose other keys are seen: no output changes by a bit."""
    rows, window, sinks = shape[3], shape[6], shape[7]
    q, k, v = inputs(shape, 81)
    lengths = lengths_of(shape)
    clean = run(capi, shape, q, k, v, lengths)
    for b, n in enumerate(lengths):
        k[b, :, n:], v[b, :, n:] = bad, bad
        first = n - rows - window + 1
        if window and first > sinks:
            k[b, :, sinks:first], v[b, :, sinks:first] = bad, bad
    again = run(capi, shape, q, k, v, lengths)
    np.testing.assert_array_equal(again.view(np.uint32), clean.view(np.uint32))


@pytest.mark.parametrize("shape", PACKED, ids=str)
def test_a_bad_key_reaches_only_the_rows_that_see_it(capi, shape):
    """NaN in a key, NaN and infinities in values: the rows of the same tile that do not
    see them stay as they are, to the bit, and the others are not finite, of a value in its
    feature alone."""
    batch, heads, kv, rows, cols, d, window, sinks = shape
    q, k, v = inputs(shape, 82)
    clean = run(capi, shape, q, k, v)
    b, where = batch - 1, cols - rows // 2
    seen = cases.visible(rows, cols, cols, window or None, sinks)[:, where]
    assert seen.any() and not seen.all()
    mine = np.zeros(clean.shape, bool)
    mine[b, :heads // kv] = seen[None, :, None]
    kk = k.copy()
    kk[b, 0, where, 5] = np.nan
    got = run(capi, shape, q, kk, v)
    assert np.isnan(got[mine]).all()
    np.testing.assert_array_equal(got[~mine].view(np.uint32), clean[~mine].view(np.uint32))
    for value in (np.nan, np.inf, -np.inf):
        vv = v.copy()
        vv[b, 0, where, 7] = value
        got = run(capi, shape, q, k, vv)
        hit = mine.copy()
        hit[..., [f for f in range(d) if f != 7]] = False
        assert not np.isfinite(got[hit]).any() and (not np.isnan(value) or np.isnan(got[hit]).all())
        rest = ~mine
        np.testing.assert_array_equal(got[rest].view(np.uint32), clean[rest].view(np.uint32))
        expected, bound = plain(shape, q, k, v, np.full(batch, cols), b, 0)
        others = [f for f in range(d) if f != 7]
        assert (np.abs(got[b, 0][:, others] - expected[:, others]) <= bound).all()


@pytest.mark.parametrize("shape", PACKED, ids=str)
def test_sequences_of_every_length(capi, shape):
    """No keys, one, fewer than queries, and all of them, in one call: rows that see nothing
    are zeros."""
    batch, heads, kv, rows, cols, d, window, sinks = shape
    for first in (0, 1, 65, rows - 1, cols):
        lengths = np.full(batch, cols)
        lengths[0] = lengths[-1] = first
        if batch > 3:
            lengths[1:3] = 0, 64
        q, k, v = inputs(shape, 83)
        got = run(capi, shape, q, k, v, lengths)
        for b, h in some_heads(shape)[:2]:
            expected, bound = plain(shape, q, k, v, lengths, b, h)
            assert (np.abs(got[b, h] - expected) <= bound).all(), (first, b, h)
        assert (got[0, :, :max(rows - first, 0)] == 0).all()


@pytest.mark.parametrize("shape", [(1, 1, 1, 1030, 0, 64, 0, 0), (43, 2, 2, 257, 0, 128, 9, 4), (128, 1, 1, 300, 0, 80, 70, 2)],
                         ids=str)
def test_no_keys_at_all(capi, shape):
    batch, heads, kv, rows, cols, d, window, sinks = shape
    q = capi.DeviceArray.from_numpy(np.ones((batch, heads, rows, d), np.float32))
    out = capi.DeviceArray.from_numpy(np.full((batch, heads, rows, d), 7, np.float32))
    desc = capi.window_attention_desc(batch, heads, kv, rows, 0, d, window=window, sinks=sinks)
    capi.window_attention(q.ptr, None, None, out.ptr, desc, workspace=capi.DeviceBuffer(1 << 20))
    capi.synchronize()
    assert (out.numpy() == 0).all()


def token_major(x, gap):
    y = np.full((x.shape[0], x.shape[2], x.shape[1], x.shape[3] + gap), np.float32(7))
    y[..., :x.shape[3]] = x.transpose(0, 2, 1, 3)
    return y


@pytest.mark.parametrize("shape", PACKED, ids=str)
def test_strides_of_packed_prompts(capi, shape):
    """Token-major tensors with gaps: the same bits as contiguous ones, nothing written
    between rows, and with less workspace than the tiles take right as well."""
    batch, heads, kv, rows, cols, d, window, sinks = shape
    q, k, v = inputs(shape, 84)
    lengths = lengths_of(shape)
    clean = run(capi, shape, q, k, v, lengths)
    qt, kt, vt, ot = token_major(q, 4), token_major(k, 8), token_major(v, 0), token_major(np.zeros_like(q), 12)
    dq, dk, dv, dn = (capi.DeviceArray.from_numpy(x) for x in (qt, kt, vt, lengths.astype(np.int32)))
    desc = capi.window_attention_desc(batch, heads, kv, rows, cols, d, window=window, sinks=sinks, lengths=dn.ptr,
                                      q_strides=strides(qt), k_strides=strides(kt), v_strides=strides(vt), out_strides=strides(ot))
    whole = capi.window_attention_workspace(desc)
    for part in (1.0, 0.9, 0.1):
        out = capi.DeviceArray.from_numpy(ot)
        capi.window_attention(dq.ptr, dk.ptr, dv.ptr, out.ptr, desc, workspace=capi.Workspace(whole.address, int(whole.nbytes * part)))
        capi.synchronize()
        got = out.numpy()
        np.testing.assert_array_equal(got[..., d:], ot[..., d:])
        result = np.ascontiguousarray(got[..., :d].transpose(0, 2, 1, 3))
        if part == 1.0:
            np.testing.assert_array_equal(result.view(np.uint32), clean.view(np.uint32))
        for b, h in some_heads(shape)[:2]:
            expected, bound = plain(shape, q, k, v, lengths, b, h)
            assert (np.abs(result[b, h] - expected) <= bound).all(), (part, b, h)


# ------------------------------------------------------------------ the 4-bit cache
@pytest.mark.parametrize("heads,kv,rows", [(2, 2, 1), (8, 2, 1), (4, 2, 20)])
@pytest.mark.parametrize("features", [32, 64, 128])
def test_cache_attention_strides_and_workspaces(capi, features, heads, kv, rows):
    """Token-major queries and outputs with gaps, every workspace from none to all."""
    rng = np.random.default_rng(85)
    batch, cols, window, sinks = 2, 5000, 4200, 5
    lengths = [4900, 2500]
    q, k, v = f32(rng, batch, heads, rows, features), f32(rng, batch, kv, cols, features), f32(rng, batch, kv, cols, features)
    keys, values = cases.cache_rows(k), cases.cache_rows(v)
    expected, bound = cases.attention(q, cases.cache_values(keys, features), cases.cache_values(values, features), lengths,
                                      window, sinks, features ** -0.5)
    qt, ot = token_major(q, 8), token_major(np.zeros_like(q), 4)
    dq, dk, dv, dn = (capi.DeviceArray.from_numpy(x) for x in (qt, keys, values, np.array(lengths, np.int32)))
    desc = capi.window_attention_desc(batch, heads, kv, rows, cols, features, window=window, sinks=sinks, lengths=dn.ptr,
                                      q_strides=strides(qt), out_strides=strides(ot))
    whole = capi.window_attention_workspace(desc, cache=True)
    for part in (0.0, 0.2, 0.6, 1.0):
        out = capi.DeviceArray.from_numpy(ot)
        ws = capi.Workspace(whole.address, int(whole.nbytes * part)) if part else None
        capi.cache4_attention(dq.ptr, dk.ptr, dv.ptr, out.ptr, desc, workspace=ws)
        capi.synchronize()
        got = out.numpy()
        np.testing.assert_array_equal(got[..., features:], ot[..., features:])
        assert (np.abs(got[..., :features].transpose(0, 2, 1, 3) - expected) <= bound).all(), part


@pytest.mark.parametrize("heads,rows", [(2, 1), (8, 3)])
def test_cache_attention_lengths_out_of_range(capi, heads, rows):
    """A negative length counts as none, one past the capacity as all of it, and both are flagged."""
    rng = np.random.default_rng(86)
    features, cols = 64, 300
    q, k, v = f32(rng, 3, heads, rows, features), f32(rng, 3, 2, cols, features), f32(rng, 3, 2, cols, features)
    keys, values = cases.cache_rows(k), cases.cache_rows(v)
    flag = ctypes.c_void_p()
    capi.check(capi.lib().tcx_hip_flag_acquire(ctypes.byref(flag)))
    for given, counted, flagged in (([-5, cols + 1, 20], [0, cols, 20], 1), ([0, cols, 20], [0, cols, 20], 0),
                                    ([2 ** 31 - 1, -2 ** 31, 7], [cols, 0, 7], 1)):
        ctypes.c_int32.from_address(flag.value).value = 0
        dq, dk, dv, dn = (capi.DeviceArray.from_numpy(x) for x in (q, keys, values, np.array(given, np.int32)))
        out = capi.DeviceArray.from_numpy(np.full_like(q, 7))
        desc = capi.window_attention_desc(3, heads, 2, rows, cols, features, lengths=dn.ptr, flag=flag.value)
        capi.cache4_attention(dq.ptr, dk.ptr, dv.ptr, out.ptr, desc)
        capi.synchronize()
        expected, bound = cases.attention(q, cases.cache_values(keys, features), cases.cache_values(values, features), counted,
                                          None, 0, features ** -0.5)
        assert (np.abs(out.numpy() - expected) <= bound).all()
        assert ctypes.c_int32.from_address(flag.value).value == flagged
    capi.lib().tcx_hip_flag_release(flag)
