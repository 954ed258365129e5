"""The 8-bit rows' and products' checks that need no GPU: what the C ABI refuses and
what it answers about sizes, the plain form against itself, and the Python
functions' arguments."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import block8_cases as cases
import tensorcx_hip_capi as capi

# Aligned host memory: a refused or empty call never touches it.
_MEMORY = (ctypes.c_char * 256)()
ADDRESS = (ctypes.addressof(_MEMORY) + 15) // 16 * 16


def refused(call, *args, **kwargs):
    with pytest.raises(capi.HipError) as error:
        call(*args, **kwargs)
    assert error.value.code == capi.TCX_INVALID_ARGUMENT, error.value


def test_words():
    for features in (0, 1, 127, 128, 129, 512, 513, 4096, 11264):
        blocks = -(-features // 128)
        assert capi.block8_words(features) == (32 * blocks, -(-blocks // 4))
    assert capi.block8_words(-1) == (0, 0)


@pytest.mark.parametrize("name", ["quantise8", "dequantise8"])
def test_rows_refuse(name):
    def call(a=ADDRESS, b=ADDRESS, c=ADDRESS, rows=2, features=5, stride=0):
        getattr(capi, name)(a, b, c, rows, features, stride, s=0)
    for change in ({"rows": -1}, {"features": -1}, {"features": 1 << 30}, {"rows": 1 << 31}, {"rows": 1 << 25, "features": 1 << 15},
                   {"stride": -8}, {"a": None}, {"b": None}, {"c": None}, {"a": ADDRESS + 2}, {"b": ADDRESS + 2},
                   {"c": ADDRESS + 2}, {"b" if name == "quantise8" else "a": ADDRESS + 4}):
        refused(call, **change)
    if name == "dequantise8":
        refused(call, stride=4)  # rows that overlap
    call(rows=0, a=None, b=None, c=None)
    call(features=0, a=None, b=None, c=None)


def test_norm_refuses():
    def call(x=ADDRESS, codes=ADDRESS, scales=ADDRESS, rows=2, features=5, epsilon=1e-5, residual=None, weight=None, total=None,
             **strides):
        capi.rmsnorm8(x, codes, scales, capi.rmsnorm8_desc(rows, features, epsilon, **strides), residual=residual, weight=weight,
                      sum=total, s=0)
    for change in ({"rows": -1}, {"features": -1}, {"features": 1 << 30}, {"rows": 1 << 31}, {"epsilon": -1e-5},
                   {"epsilon": float("nan")}, {"epsilon": float("inf")}, {"x_stride": -1}, {"residual_stride": -1},
                   {"sum_stride": -1}, {"x": None}, {"codes": None}, {"scales": None}, {"x": ADDRESS + 2}, {"codes": ADDRESS + 4},
                   {"scales": ADDRESS + 2}, {"residual": ADDRESS + 2}, {"weight": ADDRESS + 1}, {"total": ADDRESS + 2},
                   {"total": ADDRESS, "sum_stride": 4}):
        refused(call, **change)
    call(rows=0, x=None, codes=None, scales=None)
    call(features=0, x=None, codes=None, scales=None)
    assert capi.lib().tcx_hip_rmsnorm8(ADDRESS, None, None, None, ADDRESS, ADDRESS, None, None) == capi.TCX_INVALID_ARGUMENT


SPACE = capi.Workspace(ADDRESS, 1 << 30)


@pytest.mark.parametrize("gated", [False, True])
def test_products_refuse(gated):
    def call(x=ADDRESS, xs=ADDRESS, w=ADDRESS, ws=ADDRESS, out=ADDRESS, scales=ADDRESS, rows=2, features=200, outputs=5, workspace=SPACE,
             raw=None, **more):
        desc = capi.linear8_desc(rows, features, outputs, **more)
        if raw is not None:
            desc.activation = raw
        if gated:
            capi.gated_linear8(x, xs, w, ws, out, scales, desc, workspace=workspace, s=0)
        else:
            capi.linear8(x, xs, w, ws, out, desc, workspace=workspace, s=0)
    for change in ({"rows": -1}, {"features": -1}, {"outputs": -1}, {"rows": 1 << 30}, {"features": 1 << 22}, {"outputs": 1 << 29},
                   {"x": None}, {"xs": None}, {"w": None}, {"ws": None}, {"out": None}, {"x": ADDRESS + 4}, {"w": ADDRESS + 8},
                   {"xs": ADDRESS + 2}, {"ws": ADDRESS + 1}, {"out": ADDRESS + 2}, {"bias": ADDRESS + 2}, {"raw": 3}, {"raw": -1},
                   {"out_stride": -1}, {"out_stride": 4}, {"workspace": capi.Workspace(ADDRESS + 4, 1 << 30)}):
        refused(call, **change)
    if gated:
        for change in ({"scales": None}, {"scales": ADDRESS + 2}, {"out": ADDRESS + 4}, {"out_stride": 5}):
            refused(call, **change)
        wanted = capi.linear8_workspace_bytes(capi.linear8_desc(2, 2000, 5), True)
        assert wanted > 0
        for workspace in (None, capi.Workspace(ADDRESS, wanted - 1)):
            refused(call, features=2000, workspace=workspace)
    nothing = dict(x=None, xs=None, w=None, ws=None, out=None, scales=None, workspace=None)
    call(rows=0, **nothing)
    call(outputs=0, **nothing)
    with pytest.raises(KeyError):
        capi.linear8_desc(1, 1, 1, activation="tanh")
    name = "tcx_hip_gated_linear8" if gated else "tcx_hip_linear8"
    pointers = [ADDRESS] * (6 if gated else 5)
    assert getattr(capi.lib(), name)(*pointers, None, None, 0, None) == capi.TCX_INVALID_ARGUMENT


@pytest.mark.parametrize("gated", [False, True])
def test_workspace_queries(gated):
    wanted = lambda *sizes: capi.linear8_workspace_bytes(capi.linear8_desc(*sizes), gated)
    assert wanted(0, 128, 5) == 0 and wanted(5, 128, 0) == 0 and wanted(-1, 128, 5) == 0 and wanted(5, 1 << 23, 5) == 0
    assert capi.linear8_workspace(capi.linear8_desc(0, 128, 5), gated) is None
    assert getattr(capi.lib(), f"tcx_hip_{'gated_' if gated else ''}linear8_workspace_bytes")(None) == 0
    for rows in (1, 16, 100, 4096):  # what it takes stays within a few results of float32
        assert wanted(rows, 4096, 4096) <= 64 * rows * 4096 * 4 * (2 if gated else 1)


def test_plain_form():
    """The plain form against itself: codes at most half a step off, borders, ties."""
    v = cases.code_values()
    finite = v[np.isfinite(v)]
    assert finite.max() == 448 and np.isnan(v).sum() == 2 and len(np.unique(finite)) == 253
    assert np.array_equal(cases.round_to_code(finite), finite)
    between = np.sort(np.unique(np.abs(finite)))
    middle = (between[1:] + between[:-1]) / 2
    even = np.where(np.arange(len(middle)) % 2 == 0, between[:-1], between[1:])  # codes count up, so ties go to even ones
    assert np.array_equal(cases.round_to_code(middle), even)
    for top, e in ((448, 0), (np.nextafter(np.float32(448), np.float32(900)), 1), (449, 1), (1.75, -8), (1.76, -7), (1, -8), (0, -100),
                   (2.0 ** -130, -100), (3.4028234663852886e38, 120)):
        assert cases.exponents_of(np.array([float(top)]))[0] == e, top
    rng = np.random.default_rng(4)
    x = (rng.normal(size=(30, 300)) * 10.0 ** rng.integers(-20, 20, (30, 1))).astype(np.float32)
    units, e = cases.quantise(x)
    off = np.abs((units * 2.0 ** e[..., None]).reshape(30, -1)[:, :300] - x)
    assert (off <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * 2.0 ** np.repeat(e, 128, -1)[:, :300])).all()


def test_python_arguments():
    import tensorcx as cx
    x, n = cx.zeros((3, 128)), cx.zeros((3, 32), dtype="int32")
    s = cx.zeros((3, 1), dtype="int32")
    for call in (lambda: cx.hip.quantise8(x), lambda: cx.hip.rmsnorm8(x), lambda: cx.hip.dequantise8((n, s)),
                 lambda: cx.hip.linear8((n, s), (n, s)), lambda: cx.hip.gated_linear8((n, s), (n, s))):
        with pytest.raises(NotImplementedError):  # host tensors: the device computes
            call()
    for call in (lambda: cx.hip.quantise8(1), lambda: cx.hip.rmsnorm8(x, 3), lambda: cx.hip.dequantise8(n),
                 lambda: cx.hip.dequantise8((n, 3)), lambda: cx.hip.linear8((n, s), n), lambda: cx.hip.linear8([n, s], (n, s)),
                 lambda: cx.hip.gated_linear8((n, s), (n, s), 4)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: cx.hip.dequantise8((x, s)), lambda: cx.hip.dequantise8((n, n)), lambda: cx.hip.linear8((n, s), (s, s))):
        with pytest.raises(ValueError):
            call()
