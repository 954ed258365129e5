"""GPU tests of 8-bit rows and products at the ends of the format: weights next to
float32's largest value and past it, rows of which a norm makes no numbers."""

from __future__ import annotations

import numpy as np
import pytest

import block8_cases as cases
from conftest import require_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cx():
    require_gpu()
    import tensorcx
    return tensorcx


def hip(cx, a):
    return cx.tensor(a, device="hip")


def f32(rng, *shape):
    return rng.normal(size=shape).astype(np.float32)


def words(pair):
    codes, scales = (t.numpy() for t in pair)
    return codes.reshape(-1, codes.shape[-1]), scales.reshape(-1, scales.shape[-1])


CODES = {value: code for code, value in enumerate(cases.code_values()[:127])}  # of what is not negative


def coded(rng, rows, blocks, exponents):
    """Rows of random finite codes of either sign whose blocks have the given exponents."""
    codes = rng.integers(0, 127, (rows, blocks * 128)).astype(np.uint8) | (rng.integers(0, 2, (rows, blocks * 128)) << 7).astype(np.uint8)
    return codes, np.broadcast_to(exponents, (rows, blocks)).copy()


# One unit of four blocks and several, eight and more units with waves that have none in the last
# turn, in one to three turns; few rows and more, for the tiles.
@pytest.mark.parametrize("blocks", [1, 2, 4, 5, 8, 29, 33, 36, 68, 75])
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 40])
def test_linear_of_weights_next_to_the_largest(cx, rows, blocks):
    """Blocks of the largest exponent, whose values are finite, beside ordinary ones whose
    codes are large: the products are those of the values, on every way."""
    rng = np.random.default_rng(blocks)
    outputs = 50
    x_codes, x_exponents = coded(rng, rows, blocks, -100)
    w_codes, w_exponents = coded(rng, outputs, blocks, 0)
    for row in range(outputs):  # the largest in one block of the last unit, but not in its last block if there are more
        at = (blocks - 1) // 4 * 4 + row % ((blocks - 1) % 4 + 1)
        if at == blocks - 1 and blocks > 1:
            at = max(blocks - 2, 0)
        w_exponents[row, at] = 120
        here = slice(at * 128, at * 128 + 128)
        w_codes[row, here] = rng.integers(0, CODES[224.0] + 1, 128) | rng.integers(0, 2, 128) << 7
        w_codes[row, -128 + row] = CODES[448.0] if at != blocks - 1 else CODES[224.0]
    pairs = [cases.pack(x_codes, x_exponents), cases.pack(w_codes, w_exponents)]
    xv, wv = (cases.values(*p) for p in pairs)
    expected, off = cases.product(xv, wv)
    assert np.abs(wv).max() < 2.0 ** 128 and np.abs(expected).max() < 1e30
    got = cx.hip.linear8(*(tuple(hip(cx, t) for t in p) for p in pairs)).numpy()
    error = np.abs(got - expected)
    assert (error <= off + 2.0 ** -126).all(), f"off by up to {np.nanmax(error / np.maximum(off, 1e-300)):.3g} of the bound, {np.isnan(got).sum()} NaN"


@pytest.mark.parametrize("blocks", [1, 4, 9, 36, 75])
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 40])
def test_linear_of_weights_past_the_largest(cx, rows, blocks):
    """A code that stands for 2^128 is infinite: its column is infinite where it meets no
    zero, with the sign of the other factor, on every way."""
    rng = np.random.default_rng(blocks)
    outputs = 20
    x = (np.abs(f32(rng, rows, blocks * 128)) + 1) * np.where(rng.integers(0, 2, (rows, 1)), 1, -1)
    w_codes, w_exponents = coded(rng, outputs, blocks, 0)
    w_codes[::2, -128:] = CODES[1.0]
    w_codes[::2, -5], w_exponents[::2, -1] = CODES[256.0], 120
    x_pair = cx.hip.quantise8(hip(cx, x.astype(np.float32)))
    got = cx.hip.linear8(x_pair, tuple(hip(cx, t) for t in cases.pack(w_codes, w_exponents))).numpy()
    np.testing.assert_array_equal(got[:, ::2], np.sign(x[:, :1]) * np.full((rows, outputs // 2), np.inf, np.float32))
    expected, off = cases.product(cases.values(*words(x_pair)), cases.values(*cases.pack(w_codes[1::2], w_exponents[1::2])))
    assert (np.abs(got[:, 1::2] - expected) <= off).all()


# Rows that one wave holds, each number of groups a wave holds, and rows read twice; the last
# block partly filled, alone in its group and not.
@pytest.mark.parametrize("features", [1, 300, 1000, 1537, 5000, 8321, 16385, 32700, 33001, 70001])
@pytest.mark.parametrize("weight", [False, True])
def test_rmsnorm_leaves_zeros_behind_the_last_feature(cx, features, weight):
    """Codes behind the last feature are zeros whatever the row's norm is: of a NaN, of
    an infinity, of zeros with no epsilon (zero over zero); the row itself goes by the formula."""
    rng = np.random.default_rng(features)
    x = f32(rng, 5, features)
    x[1, features // 2], x[2, 0], x[3] = np.nan, -np.inf, 0
    w = hip(cx, 1 + 0.3 * f32(rng, features)) if weight else None
    for given in ({}, {"residual": hip(cx, np.zeros_like(x))}):
        codes, scales, *_ = cx.hip.rmsnorm8(hip(cx, x), w, eps=0.0, **given)
        c, e = cases.unpack(*words((codes, scales)))
        assert (c[:, features:] == 0).all(), f"rows {np.flatnonzero((c[:, features:] != 0).any(1)).tolist()}"
        got = cases.values(*words((codes, scales)))[:, :features]
        assert np.isnan(got[1]).all() and np.isnan(got[2, 0]) and (got[2, 1:] == 0).all() and np.isnan(got[3]).all()
        assert np.isfinite(got[[0, 4]]).all()
