"""Fused hip kernels reached through BackendOpClass::kKernel.

These run the built-in static-library kernels of HipBackend. "linear_bias_act"
and "bias_act": act(x @ weight^T + bias) in one GEMM epilogue, and act(x + bias)
in one pass. activation is "none", "silu" or "gelu"; results equal linear()
followed by silu()/gelu() up to the exp/tanh implementation.

The others are the operators of a decoding loop:

* ``window_attention``: attention in which a query sees a window of the last
  keys and a few first ones, with query heads that share a key head;
* ``new_cache``, ``cache_store``, ``cache_load`` and ``cache_attention``: keys and
  values held in 4 bits, 32 features to a low end and a step, and the same
  attention over them;
* ``beam_select`` and ``beam_reorder``: beam search's choice over beams and
  vocabulary, and the states of the chosen beams.

They allocate their outputs and what workspace they use, and return when the
result is there. Loops that keep buffers, run ahead or capture graphs call the C
ABI's functions of the same names (``tensorcx_hip_capi``), which do neither.
"""

from __future__ import annotations

import operator
import struct

import numpy as np

_ACT = {"none": 0, "silu": 1, "gelu": 2}


def _act(name: str) -> int:
    if name not in _ACT:
        raise ValueError(f"unknown activation {name!r}")
    return _ACT[name]


def linear_act(input, weight, bias, activation: str = "silu"):
    from . import Tensor, _core, _hip
    x, w, b = _hip(input, weight, bias, name="linear_act")
    return Tensor(_core.linear_act(x, w, b, _act(activation)))


def bias_act(input, bias, activation: str = "silu"):
    from . import Tensor, _core, _hip
    x, b = _hip(input, bias, name="bias_act")
    return Tensor(_core.bias_act(x, b, _act(activation)))


def _count(value, name: str, least: int) -> int:
    """value as an int of at least `least` that fits 32 bits."""
    if isinstance(value, (bool, np.bool_)):
        raise TypeError(f"{name} must be an integer")
    try:
        number = operator.index(value)
    except TypeError:
        raise TypeError(f"{name} must be an integer") from None
    if number < least:
        raise ValueError(f"{name} must be at least {least}")
    if number >= 2**32:
        raise ValueError(f"{name} must be below 2^32")
    return number


def _rank4(tensor, name: str) -> tuple[int, ...]:
    if len(tensor.shape) != 4:
        raise ValueError(f"{name} must have rank 4")
    return tensor.shape


def _scale_bits(scale, features: int) -> int:
    """The float32 bits of the scale (1 / sqrt(features) for None)."""
    if scale is None:
        scale = features ** -0.5 if features else 1.0
    elif isinstance(scale, (bool, np.bool_)) or not isinstance(scale, (int, float, np.integer, np.floating)):
        raise TypeError("attention scale must be a real scalar")
    try:
        with np.errstate(over="ignore"):
            narrowed = np.float32(float(scale))
    except OverflowError:
        raise ValueError("attention scale is out of range") from None
    if not np.isfinite(narrowed) or (float(scale) != 0 and narrowed == 0):
        raise ValueError("attention scale must be finite and representable as float32")
    return struct.unpack("<I", struct.pack("<f", narrowed))[0]


def _attend(entry: str, query, key, value, lengths, window, sinks, scale):
    from . import Tensor, _core, _inference
    inputs = (query, key, value) + (() if lengths is None else (lengths,))
    impls = _inference(entry, *inputs)
    shape = _rank4(query, "query")
    scalars = [0 if window is None else _count(window, "window", 1), _count(sinks, "sinks", 0),
               _scale_bits(scale, shape[3])]
    out = _core.empty(list(shape), "float32")
    _core._kernel(entry, impls, scalars, [out])
    return Tensor(out)


def window_attention(query, key, value, window=None, sinks=0, *, lengths=None, scale=None):
    """Attention of query (batch, heads, rows, features) over key and value
    (batch, kv_heads, cols, features); heads is a multiple of kv_heads, features
    a multiple of 8 from 16 to 128. Sequence b has lengths[b] keys (int32; None:
    cols), and its last query stands at its last key: query i sees the keys up
    to p = lengths[b] - rows + i that are among the last ``window`` (itself
    included; None: all) or the first ``sinks``. A query that sees no key gives
    zeros; hidden keys have no influence, whatever they hold."""
    return _attend("window_attention", query, key, value, lengths, window, sinks, scale)


def new_cache(batch: int, kv_heads: int, capacity: int, features: int):
    """A zeroed 4-bit cache: int32 (batch, kv_heads, capacity, features / 8 +
    features / 32) for 32, 64 or 128 features. Keys and values have one each."""
    from . import _core, zeros
    words = _core._cache4_words(_count(features, "features", 0))
    if words == 0:
        raise ValueError("a 4-bit cache holds 32, 64 or 128 features")
    return zeros((_count(batch, "batch", 0), _count(kv_heads, "kv_heads", 0), _count(capacity, "capacity", 0), words),
                 dtype="int32", device="hip")


def cache_store(key, value, key_cache, value_cache, positions) -> None:
    """Stores key and value (batch, kv_heads, tokens, features) in the caches, in
    place: token t of sequence b in slot positions[b] + t (int32). A value is held
    as one of 16 steps between the ends of its 32 features, at most half a step
    off. Tokens without a slot are dropped, and ValueError is raised."""
    from . import _core, _inference
    k, v, kc, vc, p = _inference("cache_store", key, value, key_cache, value_cache, positions)
    _core._kernel("cache4_store", [k, v, p], [], [kc, vc])


def cache_load(cache, start: int = 0, count: int | None = None):
    """The float32 (batch, kv_heads, count, features) that slots [start, start +
    count) of a cache stand for (None: up to the capacity)."""
    from . import Tensor, _core, _inference
    (c,) = _inference("cache_load", cache)
    batch, heads, capacity, words = _rank4(cache, "cache")
    features = next((f for f in (32, 64, 128) if _core._cache4_words(f) == words), 0)
    if not features or cache.dtype != "int32":
        raise ValueError("cache_load expects an int32 cache of 32, 64 or 128 features")
    start = _count(start, "start", 0)
    count = max(capacity - start, 0) if count is None else _count(count, "count", 0)
    if start + count > capacity:
        raise ValueError("cache slots lie past the capacity")
    out = _core.empty([batch, heads, count, features], "float32")
    _core._kernel("cache4_load", [c], [start], [out])
    return Tensor(out)


def cache_attention(query, key_cache, value_cache, lengths, window=None, sinks=0, *, scale=None):
    """window_attention over 4-bit caches, of which sequence b has lengths[b]
    slots in use."""
    return _attend("cache4_attention", query, key_cache, value_cache, lengths, window, sinks, scale)


def beam_select(logits, scores, count: int, *, finished=None, eos: int | None = None):
    """(scores, beams, tokens), (batch, count) each: of the candidates (beam k,
    token v) of every sequence the best ``count`` (at most 256) by scores[b, k] +
    log_softmax(logits[b, k])[v], in descending order, for logits (batch, beams,
    vocabulary) and scores (batch, beams) of up to 64 beams. A beam's sum of
    exponentials is float32's; candidates are compared in 64 bits. Of equal scores the
    lower beam comes first, and of one beam the larger logit, then the lower token. NaN
    comes before every number, and a beam with a NaN or +inf among its logits offers
    NaN alone. A beam that is finished (bool (batch, beams)) offers the token ``eos``
    at its own score and nothing (-inf) besides."""
    from . import Tensor, _core, _inference
    if (finished is None) != (eos is None):
        raise ValueError("finished and eos come together")
    inputs = (logits, scores) + (() if finished is None else (finished,))
    impls = _inference("beam_select", *inputs)
    if len(logits.shape) != 3:
        raise ValueError("logits must have rank 3")
    shape = [logits.shape[0], _count(count, "count", 1)]
    end = 0 if eos is None else _count(eos, "eos", 0)
    if eos is not None and end >= logits.shape[2]:
        raise ValueError("eos is outside the vocabulary")
    if shape[1] > min(256, logits.shape[1] * logits.shape[2]):
        raise ValueError("count must be at most 256 and beams * vocabulary")
    outputs = [_core.empty(shape, dtype) for dtype in ("float32", "int32", "int32")]
    _core._kernel("beam_select", impls, [end], outputs)
    return tuple(Tensor(t) for t in outputs)


def beam_reorder(states, beams):
    """The states of the chosen beams: for each tensor of ``states``, whose leading
    axis counts batch * beams rows, a new one whose row b * count + n is row b *
    beams + beams[b, n] (int32 (batch, count)). One tensor gives one tensor, an
    iterable a tuple."""
    from . import Tensor, _core, _inference
    single = isinstance(states, Tensor)
    tensors = (states,) if single else tuple(states)
    if not tensors:
        raise ValueError("beam_reorder expects at least one state")
    impls = _inference("beam_reorder", *tensors, beams)
    if len(beams.shape) != 2 or any(not t.shape for t in tensors):
        raise ValueError("beams must have rank 2 and states a leading axis")
    rows = beams.shape[0] * beams.shape[1]
    outputs = [_core.empty([rows, *t.shape[1:]], t.dtype) for t in tensors]
    _core._kernel("beam_reorder", impls, [], outputs)
    results = tuple(Tensor(t) for t in outputs)
    return results[0] if single else results
