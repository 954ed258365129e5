"""Fused hip kernels reached through BackendOpClass::kKernel.

These run the built-in static-library kernels of HipBackend. "linear_bias_act"
and "bias_act": act(x @ weight^T + bias) in one GEMM epilogue, and act(x + bias)
in one pass. activation is "none", "silu" or "gelu"; results equal linear()
followed by silu()/gelu() up to the exp/tanh implementation.

Operators of a decoding loop:

* ``window_attention``: attention in which a query sees a window of the last
  keys and a few first ones, with query heads that share a key head;
* ``new_cache``, ``cache_store``, ``cache_load`` and ``cache_attention``: keys and
  values held in 4 bits, 32 features to a low end and a step, and the same
  attention over them;
* ``beam_select`` and ``beam_reorder``: beam search's choice over beams and
  vocabulary, and the states of the chosen beams.

A layer's products with 8-bit operands, rows held as codes with a power of two for
each 128 features:

* ``quantise8`` and ``dequantise8``: float32 rows to that form, and back;
* ``rmsnorm8``: a residual added, the root-mean-square norm, its output in that form;
* ``linear8``: act(x @ weight^T + bias) of activations and weights in that form, as
  float32; ``gated_linear8``: the gated half of a layer, its output in that form.

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


def _rows8(rows, name: str):
    """The codes and scales of a pair, as quantise8 makes it."""
    from . import Tensor
    if not isinstance(rows, tuple) or len(rows) != 2 or not all(isinstance(t, Tensor) for t in rows):
        raise TypeError(f"{name} must be a pair of codes and scales")
    codes, scales = rows
    if codes.dtype != "int32" or scales.dtype != "int32":
        raise ValueError(f"{name} codes and scales must be int32")
    if not codes.shape or len(scales.shape) != len(codes.shape) or codes.shape[-1] % 32 or \
            scales.shape != (*codes.shape[:-1], (codes.shape[-1] // 32 + 3) // 4):
        raise ValueError(f"{name} codes and scales do not belong together")
    return codes, scales


def _empty8(shape):
    from . import _core
    code_words, scale_words = _core._block8_words(shape[-1])
    return [_core.empty([*shape[:-1], words], "int32") for words in (code_words, scale_words)]


def _float_rows(tensor, name: str) -> None:
    if tensor.dtype != "float32":
        raise ValueError(f"{name} must be float32")
    if not tensor.shape:
        raise ValueError(f"{name} must have at least one axis")


def quantise8(input):
    """(codes, scales), int32 (..., 32 * blocks) and (..., ceil(blocks / 4)), of float32
    (..., features): each value in 8-bit floating point (four bits of exponent, three
    of mantissa), in units of a power of two that each block of 128 features has for
    itself, the least that leaves its largest value at 448 units or below (2^-100 at
    the least). Values are rounded to the nearest code, at most 2^-4 of themselves off;
    NaN and infinities become NaN."""
    from . import Tensor, _core, _inference
    (x,) = _inference("quantise8", input)
    _float_rows(input, "input")
    outputs = _empty8(input.shape)
    _core._kernel("quantise8", [x], [], outputs)
    return tuple(Tensor(t) for t in outputs)


def dequantise8(rows, features: int | None = None):
    """The float32 (..., features) that a pair of codes and scales stands for (None: as
    many features as its blocks hold)."""
    from . import Tensor, _core, _inference
    codes, scales = _rows8(rows, "rows")
    impls = _inference("dequantise8", codes, scales)
    held = 4 * codes.shape[-1]
    features = held if features is None else _count(features, "features", 0)
    if (features + 127) // 128 * 128 != held:
        raise ValueError("features do not fill the blocks of the codes")
    out = _core.empty([*codes.shape[:-1], features], "float32")
    _core._kernel("dequantise8", impls, [], [out])
    return Tensor(out)


def _epsilon_bits(eps) -> int:
    if isinstance(eps, (bool, np.bool_)) or not isinstance(eps, (int, float, np.integer, np.floating)):
        raise TypeError("eps must be a real scalar")
    try:
        with np.errstate(over="ignore"):
            narrowed = np.float32(float(eps))
    except OverflowError:
        raise ValueError("eps is out of range") from None
    if not np.isfinite(narrowed) or narrowed < 0:
        raise ValueError("eps must be finite and not negative")
    return struct.unpack("<I", struct.pack("<f", narrowed))[0]


def rmsnorm8(input, weight=None, eps: float = 1.0e-5, *, residual=None):
    """(codes, scales) of y = s / sqrt(mean(s^2) + eps) * weight over the last axis, with
    s = input + residual; with a residual (codes, scales, s). weight is (features,)."""
    from . import Tensor, _core, _inference
    inputs = (input,) + (() if residual is None else (residual,)) + (() if weight is None else (weight,))
    impls = _inference("rmsnorm8", *inputs)
    _float_rows(input, "input")
    scalars = [_epsilon_bits(eps), int(residual is not None), int(weight is not None)]
    outputs = _empty8(input.shape)
    if residual is not None:
        outputs.append(_core.empty(list(input.shape), "float32"))
    _core._kernel("rmsnorm8", impls, scalars, outputs)
    return tuple(Tensor(t) for t in outputs)


def _product8(entry: str, input, weight, bias, activation: str):
    from . import _inference
    x, w = _rows8(input, "input"), _rows8(weight, "weight")
    impls = _inference(entry, *x, *w, *(() if bias is None else (bias,)))
    if len(w[0].shape) != 2:
        raise ValueError("weight must have rank 2")
    if w[0].shape[1] != x[0].shape[-1]:
        raise ValueError("input and weight must have the same features")
    return impls, [_act(activation)], x[0].shape[:-1], w[0].shape[0]


def linear8(input, weight, bias=None, activation: str = "none"):
    """act(input @ weight^T + bias) as float32 (..., outputs) of pairs of codes and scales:
    input (..., features), weight (outputs, features). The products are exact, their
    sums float32. activation is "none", "silu" or "gelu"."""
    from . import Tensor, _core
    impls, scalars, lead, rows = _product8("linear8", input, weight, bias, activation)
    out = _core.empty([*lead, rows], "float32")
    _core._kernel("linear8", impls, scalars, [out])
    return Tensor(out)


def gated_linear8(input, weight, bias=None, activation: str = "silu"):
    """(codes, scales) of act(input @ gate^T + bias) * (input @ up^T + bias'), for weight
    rows (and biases) of gate, then as many of up."""
    from . import Tensor, _core
    impls, scalars, lead, rows = _product8("gated_linear8", input, weight, bias, activation)
    if rows % 2:
        raise ValueError("weight must have as many gate rows as up rows")
    outputs = _empty8((*lead, rows // 2))
    _core._kernel("gated_linear8", impls, scalars, outputs)
    return tuple(Tensor(t) for t in outputs)
