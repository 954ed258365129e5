"""Plain 64-bit forms of the 8-bit rows and their products, and the errors that
float32 kernels may make."""

from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24  # half a step of float32, relative
BLOCK = 128
LOWEST = -100
LARGEST = 448.0


def blocks_of(features):
    return -(-features // BLOCK)


def code_values():
    """What the 256 codes stand for, in units of their block's power of two."""
    code = np.arange(256)
    field, mantissa = code >> 3 & 15, code & 7
    size = np.where(field == 0, mantissa / 512.0, (8 + mantissa) * 2.0 ** (field - 10.0))
    size[(code & 127) == 127] = np.nan
    return np.where(code >= 128, -size, size)


def exponents_of(top):
    """The least e >= LOWEST with top <= 448 * 2^e, of float64 values that are float32's."""
    _, e = np.frexp(top)  # top = f * 2^e with f in [0.5, 1): 448 is 0.875 * 2^9
    e = e - 9 + (top > np.ldexp(0.875, e))
    return np.maximum(np.where(top == 0, LOWEST, e), LOWEST)


def round_to_code(u):
    """Finite values of at most 448 rounded to the nearest code, ties to even."""
    _, e = np.frexp(u)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.rint(u / step) * step


def quantise(x):
    """Float32 (..., features) to the values of codes (..., blocks, 128), in units, NaN for
    NaN and infinities, and the exponents (..., blocks)."""
    features = x.shape[-1]
    g = np.zeros((*x.shape[:-1], blocks_of(features) * BLOCK))
    g[..., :features] = x
    g = g.reshape(*x.shape[:-1], -1, BLOCK)
    finite = np.isfinite(g)
    e = exponents_of(np.abs(np.where(finite, g, 0)).max(-1, initial=0))
    return np.where(finite, round_to_code(np.ldexp(np.where(finite, g, 0), -e[..., None])), np.nan), e


def pack(codes, exponents):
    """uint8 codes (rows, blocks * 128) and exponents (rows, blocks) as int32 words."""
    rows, blocks = exponents.shape
    held = np.zeros((rows, -(-blocks // 4) * 4), np.uint8)
    held[:, :blocks] = exponents + 127
    return np.ascontiguousarray(codes).view(np.int32), held.view(np.int32)


def unpack(codes, scales):
    """int32 words of rows to codes as uint8 (rows, blocks * 128) and exponents (rows, blocks)."""
    blocks = codes.shape[1] // 32
    held = np.ascontiguousarray(scales).view(np.uint8).astype(int)
    assert (held[:, blocks:] == 0).all(), "bytes behind the last block's exponent are zeros"
    return np.ascontiguousarray(codes).view(np.uint8), held[:, :blocks] - 127


def values(codes, scales):
    """What int32 words of rows stand for, in 64 bits: (rows, blocks * 128)."""
    c, e = unpack(codes, scales)
    return (code_values()[c].reshape(len(c), -1, BLOCK) * 2.0 ** e[..., None]).reshape(c.shape)


def check_quantised(codes, scales, x, context=""):
    """Words against the plain form of float32 rows, exactly (a NaN's sign aside)."""
    c, e = unpack(codes, scales)
    units, exponents = quantise(x)
    assert np.array_equal(e, exponents), f"{context}: exponents differ at {np.argwhere(e != exponents)[:4].tolist()}"
    found = code_values()[c].reshape(units.shape)
    same = (found == units) | (np.isnan(found) & np.isnan(units))
    assert same.all(), f"{context}: codes differ at {np.argwhere(~same)[:4].tolist()}"
    signs = np.zeros((*x.shape[:-1], c.shape[1]), bool)
    signs[..., :x.shape[-1]] = np.signbit(x)
    signs = signs.reshape(units.shape)
    assert np.array_equal((c >= 128).reshape(units.shape)[~np.isnan(units)], signs[~np.isnan(units)]), context


def check_near(codes, scales, y, off, context=""):
    """Words of rows computed in float32 against their values y in 64 bits, computed to
    within off: an exponent goes by the block's largest value as the kernel had it, and
    a value is off by its rounding to a code as well."""
    c, e = unpack(codes, scales)
    features = y.shape[-1]
    wide = lambda a: np.pad(np.broadcast_to(a, y.shape), ((0, 0), (0, c.shape[1] - features))).reshape(len(c), -1, BLOCK)
    g, d = wide(y), wide(off)
    low = exponents_of(np.maximum(np.abs(g) - d, 0).max(-1))
    high = exponents_of((np.abs(g) + d).max(-1))
    assert ((e >= low) & (e <= high)).all(), f"{context}: exponents {np.argwhere((e < low) | (e > high))[:4].tolist()}"
    found = code_values()[c].reshape(g.shape) * 2.0 ** e[..., None]
    bound = d + np.maximum(2.0 ** -4 * (np.abs(g) + d), 2.0 ** -10 * 2.0 ** e[..., None])
    far = np.abs(found - g) > bound
    assert not far.any(), f"{context}: values differ at {np.argwhere(far)[:4].tolist()}"
    assert (c[:, features:] == 0).all(), f"{context}: codes behind the last feature"


def activate(x, name):
    if name == "silu":
        return x / (1 + np.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1 + np.tanh(0.7978845608028654 * (x + 0.044715 * x ** 3)))
    return x


def product(x, w, bias=None, activation="none"):
    """act(x w^T + bias) of values in 64 bits, and how far float32 may be off: exact
    products in a sum of K terms in any order, each addition off by a step (2 EPS) of
    what it sums at most, which is no more than the sum of the sizes; one more for the
    bias. The slopes of the activations stay below 1.2 and their own float32 steps (a
    dozen roundings, and the exponential's or tanh's of arguments off by a few EPS of
    themselves, which reach the result at most times |v| exp(-|v|) < 1) are below 32
    EPS of |v| + 1."""
    size = np.abs(x) @ np.abs(w).T
    v = x @ w.T
    off = 2 * EPS * (x.shape[1] + 2) * size
    if bias is not None:
        v = v + bias
        off = off + EPS * (np.abs(v) + off)
    if activation != "none":
        off = 1.2 * off + 32 * EPS * (np.abs(v) + 1)
    return activate(v, activation), off


def rmsnorm(x, residual, weight, eps):
    """The sum as float32 has it, the norm of that in 64 bits, and how far float32 may be
    off: the mean of squares by the additions (a chain of at most features / 64 + 64 in
    a lane, then lanes and waves) and a few roundings, half of that in its root."""
    s = x if residual is None else x + residual
    t = s.astype(np.float64)
    y = t / np.sqrt((t * t).mean(-1, keepdims=True) + float(np.float32(eps)))
    if weight is not None:
        y = y * weight
    return s, y, (x.shape[-1] / 64 + 64 + 24) * EPS * np.abs(y)
