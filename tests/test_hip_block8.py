"""GPU tests of the 8-bit rows and their products against plain 64-bit forms,
through the package and through the C ABI.

Quantised rows and what codes stand for are exact; products, norms and gated rows
have the tolerances that block8_cases derives from float32's half step."""

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


@pytest.fixture(scope="module")
def capi():
    require_gpu()
    import tensorcx_hip_capi
    return tensorcx_hip_capi


def hip(cx, a):
    return cx.tensor(a, device="hip")


def f32(rng, *shape):
    return rng.normal(size=shape).astype(np.float32)


def words(pair):
    codes, scales = (t.numpy() for t in pair)
    return codes.reshape(-1, codes.shape[-1]), scales.reshape(-1, scales.shape[-1])


def operand(cx, rng, rows, features, spread=3):
    """A quantised matrix of values of many sizes, on the GPU, and its values."""
    x = f32(rng, rows, features) * np.exp2(rng.integers(-spread, spread + 1, (rows, features)).astype(np.float32))
    pair = cx.hip.quantise8(hip(cx, x))
    return pair, cases.values(*words(pair))


ROWS = [(1, 1), (3, 3), (2, 4), (5, 127), (4, 128), (4, 129), (1, 500), (7, 512), (2, 513), (300, 1100), (37, 4096), (1, 20001)]


@pytest.mark.parametrize("shape", ROWS, ids=str)
def test_quantise(cx, shape):
    rng = np.random.default_rng(sum(shape))
    x = f32(rng, *shape) * np.exp2(rng.integers(-12, 13, shape).astype(np.float32)) * np.float32(10) ** rng.integers(-9, 9, (shape[0], 1))
    x = x.astype(np.float32)
    pair = cx.hip.quantise8(hip(cx, x))
    assert tuple(t.dtype for t in pair) == ("int32", "int32") and tuple(t.device for t in pair) == ("hip", "hip")
    cases.check_quantised(*words(pair), x, str(shape))
    back = cx.hip.dequantise8(pair, shape[1]).numpy()
    assert back.dtype == np.float32 and np.array_equal(back, cases.values(*words(pair))[:, :shape[1]])
    assert np.array_equal(cx.hip.dequantise8(pair).numpy()[:, shape[1]:], np.zeros((shape[0], -shape[1] % 128)))


def test_quantise_borders(cx):
    """Blocks whose largest value is at a power's border, ties, zeros, float32's ends."""
    rows = []
    middle = np.sort(np.abs(cases.code_values()[np.isfinite(cases.code_values())]))
    middle = np.unique(middle)
    ties = ((middle[1:] + middle[:-1]) / 2).astype(np.float32)
    for exponent in (-140, -110, -101, -100, -99, -30, 0, 7, 119):
        for top in (448.0, 447.9999, 448.00003, 464.0, 256.0, 1.0):
            row = np.zeros(256, np.float32)
            row[:len(ties)] = np.ldexp(ties * (top / 448 if top > 440 else 1), exponent)
            row[130] = np.ldexp(np.float32(top), exponent) if exponent < 119 else np.ldexp(np.float32(top), 119)
            row[5] = -row[130]
            rows.append(row)
    rows.append(np.zeros(256, np.float32))
    rows.append(np.full(256, -0.0, np.float32))
    rows.append(np.full(256, np.float32(2) ** -149))
    rows.append(np.full(256, np.float32(-3.0e38)))
    x = np.array(rows)
    cases.check_quantised(*words(cx.hip.quantise8(hip(cx, x))), x)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_quantise_what_is_no_number(cx, bad):
    """NaN and infinities become NaN and leave the rest of their block as it is."""
    x = f32(np.random.default_rng(2), 6, 700)
    x[0, 3], x[1, 600], x[2, 128:256], x[3] = bad, bad, bad, bad
    pair = cx.hip.quantise8(hip(cx, x))
    cases.check_quantised(*words(pair), x)
    assert np.array_equal(np.isnan(cx.hip.dequantise8(pair, 700).numpy()), ~np.isfinite(x))


def test_dequantise_every_code(cx):
    """Every code at exponents from end to end, exactly as float32 (infinity past it)."""
    exponents = np.array([[-100, -99, 0], [1, 60, 110], [119, 120, -5]])
    codes = np.tile(np.arange(256, dtype=np.uint8), 2)[None, :384].repeat(3, 0)
    codes[1] = 255 - codes[1]
    pair = cases.pack(codes, exponents)
    expected = cases.values(*pair)
    with np.errstate(over="ignore"):
        expected = expected.astype(np.float32)
    got = cx.hip.dequantise8(tuple(hip(cx, t) for t in pair)).numpy()
    np.testing.assert_array_equal(got, expected)


NORMS = [(1, 1), (3, 5), (2, 128), (5, 300), (1, 4096), (4, 4097), (3, 8192), (2, 10000), (2, 16385), (2, 32768), (1, 33000), (2, 70001),
         (700, 260)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("shape", NORMS, ids=str)
def test_rmsnorm(cx, shape, residual, weight):
    rng = np.random.default_rng(shape[1])
    x, r, w = f32(rng, *shape) + 0.5, 30 * f32(rng, *shape), 1 + 0.3 * f32(rng, shape[1])
    x, r, w = x.astype(np.float32), r if residual else None, w.astype(np.float32) if weight else None
    s, y, off = cases.rmsnorm(x, r, w, 1e-5)
    given = {"residual": hip(cx, r)} if residual else {}
    codes, scales, *total = cx.hip.rmsnorm8(hip(cx, x), hip(cx, w) if weight else None, **given)
    assert len(total) == residual
    if residual:
        np.testing.assert_array_equal(total[0].numpy(), s)
    cases.check_near(*words((codes, scales)), y, off, str(shape))


def test_rmsnorm_epsilon_and_axes(cx):
    """Small rows, where epsilon counts; more axes; rows of zeros."""
    rng = np.random.default_rng(6)
    x = 1e-3 * f32(rng, 2, 3, 200)
    x[1, 2] = 0
    for eps in (1e-5, 1.0, 0.25):
        codes, scales = cx.hip.rmsnorm8(hip(cx, x), eps=eps)
        assert codes.shape == (2, 3, 64) and scales.shape == (2, 3, 1)
        _, y, off = cases.rmsnorm(x.reshape(6, 200), None, None, eps)
        cases.check_near(*words((codes, scales)), y, off)


def test_rmsnorm_of_what_is_no_number(cx):
    """A NaN or an infinity makes its row NaN throughout, or (beside an infinity) zero."""
    x = f32(np.random.default_rng(6), 4, 1000)
    x[1, 5], x[2, 990] = np.nan, np.inf
    clean = words(cx.hip.rmsnorm8(hip(cx, np.where(np.isfinite(x), x, 1).astype(np.float32))))
    codes, scales = words(cx.hip.rmsnorm8(hip(cx, x)))
    got = cases.values(codes, scales)[:, :1000]
    assert np.isnan(got[1]).all() and np.isnan(got[2, 990]) and (got[2, :990] == 0).all()
    for row in (0, 3):
        assert np.array_equal(codes[row], clean[0][row]) and np.array_equal(scales[row], clean[1][row])


# rows, outputs, features: one token to many, sizes that fit no tile, long sums, few and many results
PRODUCTS = [(1, 1, 1), (1, 16, 128), (1, 100, 300), (1, 4096, 1024), (1, 257, 11264), (2, 33, 129), (3, 5, 4000), (8, 300, 1000),
            (15, 64, 513), (16, 1000, 256), (17, 129, 640), (31, 512, 1100), (32, 96, 5000), (33, 700, 384), (48, 130, 260),
            (64, 1100, 1000), (65, 65, 65), (100, 300, 8192), (127, 129, 1000), (128, 128, 128), (129, 1, 700), (200, 2000, 512),
            (256, 256, 2048), (257, 513, 385), (300, 1100, 1000), (513, 260, 100), (700, 513, 1300), (1030, 1, 128), (1500, 900, 260)]


# Sizes past those above that take each of the tiles: 64 x 64 on four and on two waves, 128 x
# 64, 128 x 128, 256 x 128 and 256 x 256, with rows, results and features that end inside one
TILES = [(250, 4001, 1000), (100, 8192, 300), (64, 20000, 200), (700, 3000, 300), (260, 16400, 129), (1025, 4100, 256), (2040, 8190, 300),
         (3900, 4000, 130), (64, 4096, 11264), (3900, 5100, 1300),
         (2, 30000, 300), (600, 12000, 300), (700, 9000, 300), (1416, 30, 6702), (35, 16925, 2764), (2189, 20, 4691),
         (614, 1878, 7432), (1524, 646, 5762), (5972, 674, 6026)]


@pytest.mark.parametrize("shape", PRODUCTS + TILES, ids=str)
def test_linear(cx, shape):
    rows, outputs, features = shape
    rng = np.random.default_rng(rows + outputs + features)
    (x, xv), (w, wv) = operand(cx, rng, rows, features), operand(cx, rng, outputs, features)
    expected, off = cases.product(xv, wv)
    got = cx.hip.linear8(x, w)
    assert got.dtype == "float32" and got.shape == (rows, outputs)
    error = np.abs(got.numpy() - expected)
    assert (error <= off).all(), f"off by up to {(error / np.maximum(off, 1e-300)).max():.3g} of the bound"


@pytest.mark.parametrize("shape", PRODUCTS + TILES, ids=str)
def test_linear_keeps_every_bit_of_whole_numbers(cx, shape):
    """Codes that stand for whole numbers, large ones beside ones, whose sums stay below
    2^24 in any order: float32 sums are exact, whatever their order."""
    rows, outputs, features = shape
    rng = np.random.default_rng(features)
    def whole(n):
        x = rng.integers(-3, 4, (n, features)).astype(np.float32)
        spots = rng.integers(0, features, (n, 8))  # eight of a row at most 240: 8 * 240 * 240 and the rest below 2^24
        np.put_along_axis(x, spots, rng.choice([240.0, -224.0, 176.0, 13.0], (n, 8)).astype(np.float32), 1)
        return x
    x, w = whole(rows), whole(outputs)
    assert 16 * 240 * 240 + features * 9 + 16 * 240 * 3 < 2 ** 24
    pairs = [cx.hip.quantise8(hip(cx, t)) for t in (x, w)]
    for pair, t in zip(pairs, (x, w)):
        kept = cases.values(*words(pair))
        assert np.array_equal(kept[:, :features], t), "these values are codes"
    got = cx.hip.linear8(*pairs).numpy()
    np.testing.assert_array_equal(got, x.astype(float) @ w.T.astype(float))


@pytest.mark.parametrize("activation", ["none", "silu", "gelu"])
@pytest.mark.parametrize("shape", [(1, 200, 300), (9, 200, 300), (40, 130, 700), (300, 200, 300), (20, 130, 9000), (1025, 4100, 256), (4100, 5000, 700)], ids=str)
def test_linear_bias_and_activation(cx, shape, activation):
    rows, outputs, features = shape
    rng = np.random.default_rng(rows)
    (x, xv), (w, wv) = operand(cx, rng, rows, features, 1), operand(cx, rng, outputs, features, 1)
    bias = f32(rng, outputs) * 10
    expected, off = cases.product(xv, wv, bias, activation)
    error = np.abs(cx.hip.linear8(x, w, hip(cx, bias), activation).numpy() - expected)
    assert (error <= off).all(), f"off by up to {(error / off).max():.3g} of the bound"


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_linear_exponents_from_end_to_end(cx, rows):
    """Blocks of every exponent in both operands; sums past float32 are infinite."""
    rng = np.random.default_rng(rows)
    features, outputs = 6 * 128, 70
    def scaled(n, low, high):
        e = rng.integers(low, high + 1, (n, 6))
        codes = rng.integers(0, 127, (n, features)).astype(np.uint8) | (rng.integers(0, 2, (n, features)) << 7).astype(np.uint8)
        pair = cases.pack(codes, e)
        return tuple(hip(cx, t) for t in pair), cases.values(*pair)
    for low, high in ((-100, -1), (-20, 20), (0, 40)):
        (x, xv), (w, wv) = scaled(rows, low, high), scaled(outputs, -high, -low)
        expected, off = cases.product(xv, wv)
        assert (np.abs(cx.hip.linear8(x, w).numpy() - expected) <= off + 2.0 ** -126).all()
    (x, xv), (w, wv) = scaled(rows, 118, 119), scaled(outputs, 118, 119)
    assert not np.isfinite(cx.hip.linear8(x, w).numpy()).any()


@pytest.mark.parametrize("rows", [1, 12, 40, 150, 3000])
def test_linear_of_what_is_no_number(cx, rows):
    """A NaN reaches its row (of a weight: its column) and nothing else."""
    rng = np.random.default_rng(rows)
    x, w = f32(rng, rows, 500), f32(rng, 90, 500)
    clean = cx.hip.linear8(cx.hip.quantise8(hip(cx, x)), cx.hip.quantise8(hip(cx, w))).numpy()
    x[rows // 2, 333], w[17, 0], w[89, 499] = np.nan, np.inf, np.nan
    got = cx.hip.linear8(cx.hip.quantise8(hip(cx, x)), cx.hip.quantise8(hip(cx, w))).numpy()
    bad = np.zeros(got.shape, bool)
    bad[rows // 2], bad[:, 17], bad[:, 89] = True, True, True
    assert np.isnan(got[bad]).all()
    # The blocks that hold a NaN take their exponents from the rest, as the clean ones do here.
    _, off = cases.product(np.abs(np.nan_to_num(x.astype(float), posinf=0)) * 1.1, np.abs(np.nan_to_num(w.astype(float), posinf=0)) * 1.1)
    assert (np.abs(got - clean)[~bad] <= 2 * off[~bad]).all()


def test_linear_of_nothing(cx):
    empty = lambda *shape: cx.zeros(shape, dtype="int32", device="hip")
    bias = hip(cx, np.array([1.0, -2.0, 3.0], np.float32))
    got = cx.hip.linear8((empty(2, 0), empty(2, 0)), (empty(3, 0), empty(3, 0)), bias, "silu").numpy()
    np.testing.assert_allclose(got, cases.activate(np.array([[1.0, -2.0, 3.0]] * 2), "silu"), rtol=32 * cases.EPS)
    assert cx.hip.linear8((empty(0, 32), empty(0, 1)), (empty(3, 32), empty(3, 1))).shape == (0, 3)
    assert cx.hip.linear8((empty(4, 32), empty(4, 1)), (empty(0, 32), empty(0, 1))).shape == (4, 0)
    codes, scales = cx.hip.gated_linear8((empty(2, 32), empty(2, 1)), (empty(0, 32), empty(0, 1)))
    assert codes.shape == (2, 0) and scales.shape == (2, 0)
    codes, scales = cx.hip.gated_linear8((empty(2, 0), empty(2, 0)), (empty(6, 0), empty(6, 0)))
    assert np.array_equal(cases.values(codes.numpy(), scales.numpy()), np.zeros((2, 128)))
    assert cx.hip.quantise8(hip(cx, np.zeros((3, 0), np.float32)))[0].shape == (3, 0)
    assert cx.hip.dequantise8((empty(0, 32), empty(0, 1)), 100).shape == (0, 100)


# rows, outputs, features
GATED = [(1, 1, 128), (1, 300, 1000), (2, 128, 256), (7, 129, 300), (16, 1100, 384), (33, 513, 640), (70, 256, 100), (129, 260, 1300),
         (300, 140, 513), (520, 900, 256), (1100, 3000, 129), (2050, 1000, 384), (2300, 2570, 200),
         (64, 11264, 300), (100, 3000, 1000), (260, 2000, 700), (600, 3000, 300), (130, 700, 8000), (40, 300, 9000), (4000, 2600, 200),
         (7, 129, 2000), (16, 1100, 1500), (64, 11264, 1500), (600, 700, 6000), (1000, 4000, 600),
         (1188, 194, 1064), (359, 1391, 6565), (429, 1155, 4374), (972, 2055, 6498)]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("shape", GATED, ids=str)
def test_gated_linear(cx, shape, bias):
    rows, outputs, features = shape
    rng = np.random.default_rng(outputs)
    activation = ("silu", "gelu", "none")[rows % 3]
    (x, xv), (w, wv) = operand(cx, rng, rows, features, 1), operand(cx, rng, 2 * outputs, features, 1)
    b = f32(rng, 2 * outputs) if bias else None
    pair = cx.hip.gated_linear8(x, w, hip(cx, b) if bias else None, activation)
    gate, gate_off = cases.product(xv, wv[:outputs], b[:outputs] if bias else None, activation)
    up, up_off = cases.product(xv, wv[outputs:], b[outputs:] if bias else None)
    y = gate * up
    off = gate_off * (np.abs(up) + up_off) + np.abs(gate) * up_off + cases.EPS * np.abs(y)
    assert pair[0].shape == (rows, -(-outputs // 128) * 32)
    cases.check_near(*words(pair), y, off, str(shape))


@pytest.mark.parametrize("shape", [(3, 260, 500), (3, 260, 1000), (40, 260, 2000), (100, 260, 300), (4400, 1410, 200)], ids=str)
def test_gated_linear_of_what_is_no_number(cx, shape):
    """A NaN reaches its row (of a weight: its column), not the rest of its block, and nothing
    behind the last output."""
    rows, outputs, features = shape
    rng = np.random.default_rng(rows + features)
    x, w = f32(rng, rows, features), f32(rng, 2 * outputs, features)
    def run():
        pair = cx.hip.gated_linear8(cx.hip.quantise8(hip(cx, x)), cx.hip.quantise8(hip(cx, w)), activation="none")
        codes, scales = words(pair)
        return cases.values(codes, scales), 2.0 ** (scales.view(np.uint8).max().astype(float) - 127)
    clean, unit = run()
    x[rows // 2, 33], w[17, 0], w[outputs + 130, features - 1] = np.nan, np.inf, np.nan
    got, unit_too = run()
    bad = np.zeros(got.shape, bool)
    bad[rows // 2, :outputs], bad[:, 17], bad[:, 130] = True, True, True
    assert np.array_equal(np.isnan(got), bad) and (got[:, outputs:] == 0).all()
    # The same float32 values, each rounded by 2^-4 of itself or 2^-10 of its unit at most, in
    # blocks whose exponents may differ without the columns that are NaN now.
    most = np.maximum(np.abs(got), np.abs(clean)) / (1 - 2.0 ** -4) + 2.0 ** -10 * max(unit, unit_too)
    assert (np.abs(got - clean)[~bad] <= 2 * (2.0 ** -4 * most + 2.0 ** -10 * max(unit, unit_too))[~bad]).all()


def test_shapes_of_more_axes(cx):
    rng = np.random.default_rng(1)
    x = cx.hip.quantise8(hip(cx, f32(rng, 2, 3, 200)))
    assert x[0].shape == (2, 3, 64) and x[1].shape == (2, 3, 1)
    w, wv = operand(cx, rng, 40, 200)
    flat = cx.hip.linear8(tuple(hip(cx, t) for t in words(x)), w).numpy()
    got = cx.hip.linear8(x, w)
    assert got.shape == (2, 3, 40) and np.array_equal(got.numpy().reshape(6, 40), flat)
    codes, scales = cx.hip.gated_linear8(x, w)
    assert codes.shape == (2, 3, 32) and scales.shape == (2, 3, 1)
    one = cx.hip.quantise8(hip(cx, f32(rng, 200)))
    assert one[0].shape == (64,) and cx.hip.linear8(one, w).shape == (40,)


def test_package_refuses(cx):
    rng = np.random.default_rng(1)
    x, w = cx.hip.quantise8(hip(cx, f32(rng, 4, 200))), cx.hip.quantise8(hip(cx, f32(rng, 5, 200)))
    short = cx.hip.quantise8(hip(cx, f32(rng, 5, 100)))
    for call in (lambda: cx.hip.linear8(x, short), lambda: cx.hip.linear8(x, w, hip(cx, f32(rng, 4))),
                 lambda: cx.hip.linear8(x, w, activation="tanh"), lambda: cx.hip.gated_linear8(x, w),
                 lambda: cx.hip.linear8((x[0], w[1]), w), lambda: cx.hip.dequantise8(x, 300), lambda: cx.hip.dequantise8(x, 100),
                 lambda: cx.hip.quantise8(x[0]), lambda: cx.hip.quantise8(hip(cx, np.float32(3))),
                 lambda: cx.hip.rmsnorm8(hip(cx, f32(rng, 4, 200)), hip(cx, f32(rng, 199))),
                 lambda: cx.hip.rmsnorm8(hip(cx, f32(rng, 4, 200)), residual=hip(cx, f32(rng, 3, 200))),
                 lambda: cx.hip.rmsnorm8(hip(cx, f32(rng, 4, 200)), eps=-1.0), lambda: cx.hip.rmsnorm8(x[0]),
                 lambda: cx.hip.linear8(x, cx.hip.quantise8(hip(cx, f32(rng, 2, 5, 200))))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        cx.hip.rmsnorm8(hip(cx, f32(rng, 4, 200)), eps=True)


def test_a_layer(cx):
    """The operators as a layer of a decoding loop runs them, each stage against the plain
    form of what the stage before gave."""
    rng = np.random.default_rng(12)
    batch, width, heads, kv, d, inner = 3, 384, 6, 2, 64, 500
    hidden = f32(rng, batch, width)
    def weights(n, k):
        pair = cx.hip.quantise8(hip(cx, (f32(rng, n, k) * k ** -0.5).astype(np.float32)))
        return pair, cases.values(*words(pair))
    (qkv, qkv_v), (mix, mix_v) = weights((heads + 2 * kv) * d, width), weights(width, heads * d)
    (first, first_v), (second, second_v) = weights(2 * inner, width), weights(width, inner)
    gain = 1 + 0.1 * f32(rng, 2, width)
    key_cache, value_cache = (cx.hip.new_cache(batch, kv, 20, d) for _ in range(2))

    normed = cx.hip.rmsnorm8(hip(cx, hidden), hip(cx, gain[0]))
    _, y, off = cases.rmsnorm(hidden, None, gain[0], 1e-5)
    cases.check_near(*words(normed), y, off)
    projected = cx.hip.linear8(normed, qkv).numpy()
    expected, off = cases.product(cases.values(*words(normed)), qkv_v)
    assert (np.abs(projected - expected) <= off).all()
    q, k, v = (t.reshape(batch, -1, 1, d) for t in np.split(projected, [heads * d, (heads + kv) * d], 1))
    positions = hip(cx, np.zeros(batch, np.int32))
    cx.hip.cache_store(hip(cx, np.ascontiguousarray(k)), hip(cx, np.ascontiguousarray(v)), key_cache, value_cache, positions)
    mixed = cx.hip.cache_attention(hip(cx, np.ascontiguousarray(q)), key_cache, value_cache, hip(cx, np.ones(batch, np.int32)))
    mixed = mixed.numpy().reshape(batch, heads * d)  # one token: its own value, as the cache holds it
    packed = cx.hip.quantise8(hip(cx, mixed))
    cases.check_quantised(*words(packed), mixed)
    out = cx.hip.linear8(packed, mix)
    expected, off = cases.product(cases.values(*words(packed)), mix_v)
    assert (np.abs(out.numpy() - expected) <= off).all()
    codes, scales, total = cx.hip.rmsnorm8(out, hip(cx, gain[1]), residual=hip(cx, hidden))
    s, y, off = cases.rmsnorm(out.numpy(), hidden, gain[1], 1e-5)
    np.testing.assert_array_equal(total.numpy(), s)
    cases.check_near(*words((codes, scales)), y, off)
    gated = cx.hip.gated_linear8((codes, scales), first)
    xv = cases.values(*words((codes, scales)))
    gate, gate_off = cases.product(xv, first_v[:inner], None, "silu")
    up, up_off = cases.product(xv, first_v[inner:])
    off = gate_off * (np.abs(up) + up_off) + np.abs(gate) * up_off + cases.EPS * np.abs(gate * up)
    cases.check_near(*words(gated), gate * up, off)
    final = cx.hip.linear8(gated, second).numpy()
    expected, off = cases.product(cases.values(*words(gated)), second_v)
    assert (np.abs(final - expected) <= off).all()
