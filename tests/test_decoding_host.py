"""The decoding operators' checks that need no GPU: what the C ABI refuses and
what it answers about sizes, and the Python functions' arguments."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import decoding_cases as cases
import tensorcx_hip_capi as capi

# Aligned host memory: a refused or empty call never touches it.
_MEMORY = (ctypes.c_char * 256)()
ADDRESS = (ctypes.addressof(_MEMORY) + 15) // 16 * 16


def refused(call, *args, **kwargs):
    with pytest.raises(capi.HipError) as error:
        call(*args, **kwargs)
    assert error.value.code == capi.TCX_INVALID_ARGUMENT, error.value


def attend(desc, q=ADDRESS, k=ADDRESS, v=ADDRESS, out=ADDRESS, cache=False, workspace=None):
    call = capi.cache4_attention if cache else capi.window_attention
    call(q, k, v, out, desc, workspace=workspace, s=0)


SIZES = {"batch": 2, "heads": 4, "kv_heads": 2, "rows": 1, "cols": 64, "features": 64}


@pytest.mark.parametrize("cache", [False, True])
@pytest.mark.parametrize("change", [
    {"batch": -1}, {"heads": -4}, {"kv_heads": 0}, {"kv_heads": 3}, {"rows": -1}, {"cols": -1}, {"features": 0},
    {"features": 12}, {"features": 136}, {"features": 256}, {"cols": 1 << 30}, {"rows": 1 << 29}, {"batch": 1 << 29}])
def test_attention_refuses_sizes(cache, change):
    refused(attend, capi.window_attention_desc(**{**SIZES, **change}), cache=cache)


@pytest.mark.parametrize("cache", [False, True])
@pytest.mark.parametrize("options", [{"window": -1}, {"sinks": -1}, {"scale": float("inf")}, {"scale": float("nan")},
                                     {"q_strides": (64, 64, -64)}, {"out_strides": (256, 64, 66)}])
def test_attention_refuses_options(cache, options):
    refused(attend, capi.window_attention_desc(**SIZES, **options), cache=cache)


def test_attention_refuses_buffers():
    desc = capi.window_attention_desc(**SIZES)
    for name in ("q", "k", "v", "out"):
        refused(attend, desc, **{name: None})
        refused(attend, desc, **{name: ADDRESS + 4})
        refused(attend, desc, cache=True, **{name: ADDRESS + 8})
    refused(attend, desc, workspace=capi.Workspace(ADDRESS + 4, 64))
    refused(attend, capi.window_attention_desc(**SIZES, k_strides=(8192, 4096, 62)))
    with pytest.raises(capi.HipError):
        capi.check(capi.lib().tcx_hip_window_attention_f32(1, 1, 1, 1, None, None, 0, None))


def test_only_float_keys_take_other_features():
    assert [f for f in range(0, 200) if capi.lib().tcx_hip_window_attention_supported(f)] == list(range(16, 129, 8))
    assert {f: capi.cache4_words(f) for f in range(-8, 300) if capi.cache4_words(f)} == {32: 5, 64: 10, 128: 20}
    refused(attend, capi.window_attention_desc(**{**SIZES, "features": 80}), cache=True)


@pytest.mark.parametrize("change", [{"batch": 0}, {"heads": 0, "kv_heads": 0}, {"rows": 0}])
@pytest.mark.parametrize("cache", [False, True])
def test_attention_of_nothing(change, cache):
    desc = capi.window_attention_desc(**{**SIZES, **change})
    attend(desc, q=None, k=None, v=None, out=None, cache=cache)
    assert capi.window_attention_workspace(desc, cache) is None


def test_workspace_follows_the_keys():
    """Few rows over many keys can use a workspace, many rows or few keys none;
    a narrow window leaves few keys."""
    def wanted(cache=False, **change):
        desc = capi.window_attention_desc(**{**SIZES, **change})
        query = "tcx_hip_cache4_attention_workspace_bytes" if cache else "tcx_hip_window_attention_workspace_bytes"
        return getattr(capi.lib(), query)(ctypes.byref(desc))
    for cache in (False, True):
        assert wanted(cache, cols=100000) > 0
        assert wanted(cache, cols=100000, window=16) == 0 or wanted(cache, cols=100000, window=16) < wanted(cache, cols=100000)
        assert wanted(cache, cols=16) == 0
        assert wanted(cache, features=12) == 0


def store(desc, key=ADDRESS, value=ADDRESS, key_cache=ADDRESS, value_cache=ADDRESS, positions=ADDRESS):
    capi.cache4_store(key, value, key_cache, value_cache, positions, desc, s=0)


def test_store_refuses():
    sizes = {"batch": 2, "kv_heads": 2, "tokens": 3, "capacity": 8, "features": 64}
    for change in ({"batch": -1}, {"kv_heads": -1}, {"tokens": -1}, {"capacity": -1}, {"features": 80}, {"features": 16},
                   {"capacity": 1 << 30}, {"tokens": 1 << 30}, {"batch": 1 << 30}, {"key_strides": (64, 64, 62)},
                   {"value_strides": (-64, 64, 64)}):
        refused(store, capi.cache4_store_desc(**{**sizes, **change}))
    desc = capi.cache4_store_desc(**sizes)
    for name in ("key", "value", "key_cache", "value_cache", "positions"):
        refused(store, desc, **{name: None})
    for name in ("key", "value", "key_cache", "value_cache"):
        refused(store, desc, **{name: ADDRESS + 4})
    for change in ({"batch": 0}, {"kv_heads": 0}, {"tokens": 0}):
        store(capi.cache4_store_desc(**{**sizes, **change}), None, None, None, None, None)


def test_load_refuses():
    def load(cache=ADDRESS, out=ADDRESS, heads=2, capacity=8, start=0, count=8, features=64):
        capi.cache4_load(cache, out, heads, capacity, start, count, features, s=0)
    for change in ({"heads": -1}, {"capacity": -1}, {"start": -1}, {"count": -1}, {"features": 48}, {"start": 1},
                   {"count": 9}, {"start": 9, "count": 0}, {"cache": None}, {"out": None}, {"cache": ADDRESS + 4},
                   {"out": ADDRESS + 8}, {"start": 2 ** 62, "count": 2 ** 62}):
        refused(load, **change)
    load(count=0, cache=None, out=None)
    load(heads=0, cache=None, out=None)


def test_select_refuses():
    def select(logits=ADDRESS, scores=ADDRESS, a=ADDRESS, b=ADDRESS, c=ADDRESS, batch=1, beams=2, vocabulary=10, count=4,
               workspace=capi.Workspace(ADDRESS, 1 << 20), **more):
        capi.beam_select(logits, scores, a, b, c, batch, beams, vocabulary, count, workspace=workspace, s=0, **more)
    for change in ({"batch": -1}, {"beams": 0}, {"beams": 65}, {"vocabulary": 0}, {"count": 0}, {"count": 21},
                   {"count": 257, "vocabulary": 1000}, {"vocabulary": 2 ** 30}, {"batch": 2 ** 30}, {"logits": None},
                   {"scores": None}, {"a": None}, {"b": None}, {"c": None}, {"workspace": None},
                   {"workspace": capi.Workspace(ADDRESS, 16)}, {"workspace": capi.Workspace(ADDRESS + 8, 1 << 20)},
                   {"finished": ADDRESS, "eos": -1}, {"finished": ADDRESS, "eos": 10}):
        refused(select, **change)
    select(batch=0)
    bytes_of = capi.lib().tcx_hip_beam_select_workspace_bytes
    assert bytes_of(1, 0, 10, 1) == 0 and 0 < bytes_of(1, 2, 10, 4) < bytes_of(4, 2, 10, 4) < bytes_of(4, 2, 100000, 4)


def test_reorder_refuses():
    def reorder(sources=(ADDRESS,), targets=(ADDRESS + 64,), row_bytes=(16,), index=ADDRESS, batch=1, beams=2, count=2):
        capi.beam_reorder(capi.beam_reorder_plan(sources, targets, row_bytes), index, batch, beams, count, s=0)
    for change in ({"batch": -1}, {"beams": -1}, {"count": -1}, {"beams": 0}, {"index": None}, {"sources": (None,)},
                   {"targets": (None,)}, {"row_bytes": (-1,)}, {"batch": 2 ** 30}, {"count": 2 ** 31}):
        refused(reorder, **change)
    with pytest.raises(ValueError):
        reorder(row_bytes=(16, 16))
    reorder(batch=0)
    reorder(count=0)
    reorder((), (), ())


def test_flag_needs_an_output():
    assert capi.lib().tcx_hip_flag_acquire(None) == capi.TCX_INVALID_ARGUMENT
    capi.lib().tcx_hip_flag_release(None)


def test_plain_cache_format():
    """The plain format against itself: values at most half a step off, ends kept."""
    rng = np.random.default_rng(3)
    for features in (32, 64, 128):
        x = (rng.normal(size=(50, features)) * 10.0 ** rng.integers(-6, 6, (50, 1)) + rng.normal(size=(50, 1)) * 5).astype(np.float32)
        rows = cases.cache_rows(x)
        assert rows.dtype == np.int32 and rows.shape == (50, capi.cache4_words(features))
        off = np.abs(cases.cache_values(rows, features) - x).reshape(50, -1, 32).max(-1)
        words = rows[:, features // 8:].copy().view(np.uint32)
        step = (words << np.uint32(16)).view(np.float32).astype(float)
        # Half a step, and the roundings of x - low and of the quotient (16 EPS each).
        assert (off <= step * (0.5 + 32 * cases.EPS) + np.abs(x).max() * 2 * cases.EPS).all()
    assert np.isnan(cases.cache_values(cases.cache_rows(np.full((1, 32), np.inf, np.float32)), 32)).all()


def test_python_arguments():
    import tensorcx as cx
    x = cx.zeros((1, 2, 3, 64))
    for call in (lambda: cx.hip.window_attention(x, x, x), lambda: cx.hip.cache_load(x),
                 lambda: cx.hip.beam_reorder(x, x), lambda: cx.hip.beam_select(x, x, 1)):
        with pytest.raises(NotImplementedError):  # host tensors: the device computes
            call()
    for call in (lambda: cx.hip.window_attention(1, x, x), lambda: cx.hip.cache_store(x, x, x, x, None),
                 lambda: cx.hip.cache_attention(x, x, x, None and x or 3), lambda: cx.hip.beam_reorder([x], 4)):
        with pytest.raises(TypeError):
            call()
    for value in (True, "1", 1.5):
        with pytest.raises(TypeError):
            cx.hip.new_cache(1, 1, value, 64)
    with pytest.raises(ValueError):
        cx.hip.new_cache(1, 1, 4, 80)
    with pytest.raises(ValueError):
        cx.hip.new_cache(1, -1, 4, 64)
    with pytest.raises(ValueError):
        cx.hip.beam_select(x, x, 1, eos=3)
    with pytest.raises(ValueError):
        cx.hip.beam_reorder([], x)
