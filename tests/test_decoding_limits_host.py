"""Limits of the decoding operators that need no GPU: workspaces of the largest sizes,
and what the Python functions say of numbers out of range."""

from __future__ import annotations

import ctypes

import pytest

import tensorcx_hip_capi as capi


def wanted(**sizes):
    return capi.lib().tcx_hip_window_attention_workspace_bytes(ctypes.byref(capi.window_attention_desc(**sizes)))


def test_workspaces_past_64_bits_are_not_asked_for():
    """Packed tiles take about as many bytes as the keys and values; where that is more
    than a size holds, no rest of it is asked for, or taken to be enough."""
    sizes = {"heads": 1, "kv_heads": 1, "rows": 1024, "features": 128}
    for batch in (2 ** 27, 2 ** 28 + 12345, 2 ** 29 - 1):
        for cols in (2 ** 29, 2 ** 30 - 1):
            assert wanted(batch=batch, cols=cols, **sizes) == 0
    # Below that it is what the tiles take.
    for batch in (1, 7, 2 ** 20):
        for cols in (64, 1000, 2 ** 20):
            keys = batch * cols * 128 * 4 * 2
            assert keys <= wanted(batch=batch, cols=cols, **sizes) <= 1.1 * keys + batch * 70000


def test_numbers_past_32_bits_are_named():
    import tensorcx as cx
    for number, words in ((2 ** 32, "below 2"), (2 ** 70, "below 2"), (-1, "at least 0")):
        with pytest.raises(ValueError, match=words):
            cx.hip.new_cache(1, 1, number, 64)
