"""GPU tests of every way to a product of 8-bit rows, each with bias and activation, against
the plain 64-bit form; and NaN on each, which reach their row or column and change nothing
else. test_block8_plan_host says that the sizes take the ways they are listed under."""

from __future__ import annotations

import numpy as np
import pytest

import block8_cases as cases
import block8_ways as ways
from conftest import require_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cx():
    require_gpu()
    import tensorcx
    return tensorcx


def hip(cx, a):
    return cx.tensor(a, device="hip")


def words(pair):
    return tuple(t.numpy() for t in pair)


def coded(rng, rows, features, low, high):
    """Random codes of either sign and exponents, zeros behind the last feature: uint8 and exponents."""
    blocks = cases.blocks_of(features)
    codes = rng.integers(0, 127, (rows, blocks * 128), np.uint8) | rng.integers(0, 2, (rows, blocks * 128), np.uint8) << 7
    codes[:, features:] = 0
    return codes, rng.integers(low, high + 1, (rows, blocks))


def operands(shape, weights):
    rows, outputs, features = shape
    rng = np.random.default_rng(rows + outputs + features)
    x, w = coded(rng, rows, features, -9, -7), coded(rng, weights, features, -13, -11)
    bias = rng.normal(size=weights).astype(np.float32)
    return x, w, bias, ("none", "silu", "gelu")[(rows + outputs) % 3]


def on_gpu(cx, codes, exponents):
    return tuple(hip(cx, t) for t in cases.pack(codes, exponents))


@pytest.mark.parametrize("way,shape", ways.flat(ways.LINEAR), ids=str)
def test_linear(cx, way, shape):
    rows, outputs, features = shape
    x, w, bias, activation = operands(shape, outputs)
    def run():
        return cx.hip.linear8(on_gpu(cx, *x), on_gpu(cx, *w), hip(cx, bias), activation).numpy()
    clean = run()
    expected, off = cases.product(cases.values(*cases.pack(*x)), cases.values(*cases.pack(*w)), bias, activation)
    error = np.abs(clean - expected)
    assert (error <= off).all(), f"off by up to {(error / off).max():.3g} of the bound"
    row, columns = rows // 2, [0, outputs // 2, outputs - 1]
    x[0][row, features - 1] = 0x7f
    w[0][columns, [0, features // 2, features - 1]] = 0xff
    got, bad = run(), np.zeros((rows, outputs), bool)
    bad[row], bad[:, columns] = True, True
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("way,shape", ways.flat(ways.GATED) + ways.flat(ways.GATED_ONE_LAUNCH), ids=str)
def test_gated_linear(cx, way, shape):
    rows, outputs, features = shape
    x, w, bias, activation = operands(shape, 2 * outputs)
    def run():
        return words(cx.hip.gated_linear8(on_gpu(cx, *x), on_gpu(cx, *w), hip(cx, bias), activation))
    clean = run()
    xv, wv = cases.values(*cases.pack(*x)), cases.values(*cases.pack(*w))
    gate, gate_off = cases.product(xv, wv[:outputs], bias[:outputs], activation)
    up, up_off = cases.product(xv, wv[outputs:], bias[outputs:])
    off = gate_off * (np.abs(up) + up_off) + np.abs(gate) * up_off + cases.EPS * np.abs(gate * up)
    cases.check_near(*clean, gate * up, off, str(shape))
    row, columns = rows // 2, [0, outputs - 1]
    x[0][row, 0] = 0x7f
    w[0][[0, 2 * outputs - 1], [features - 1, features // 2]] = 0x7f
    got, bad = run(), np.zeros((rows, outputs), bool)
    bad[row], bad[:, columns] = True, True
    values = cases.values(*got)
    assert np.array_equal(np.isnan(values[:, :outputs]), bad) and (values[:, outputs:] == 0).all()
    other = [r for r in range(rows) if r != row]
    blocks = [b for b in range(cases.blocks_of(outputs)) if b not in (0, (outputs - 1) // 128)]
    for found, kept in zip(*(map(lambda t: t.reshape(rows, -1, 128) if t.shape[1] > 4 * clean[1].shape[1] else t,
                                 cases.unpack(*pair)) for pair in (got, clean))):
        np.testing.assert_array_equal(found[np.ix_(other, blocks)], kept[np.ix_(other, blocks)])
