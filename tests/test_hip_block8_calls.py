"""GPU tests of how the 8-bit rows' and products' C ABI is called: strides and
addresses, outputs' surroundings, sums in place, with a workspace and without,
captured graphs, several streams and threads, offsets past 32 bits."""

from __future__ import annotations

import ctypes
import threading

import numpy as np
import pytest

import block8_cases as cases
from conftest import require_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    require_gpu()
    import tensorcx_hip_capi
    assert tensorcx_hip_capi.available()
    return tensorcx_hip_capi


@pytest.fixture(scope="module")
def runtime(capi):
    """The HIP runtime that the library runs on: streams and graphs."""
    with open("/proc/self/maps") as f:
        paths = {line.split()[-1] for line in f if "libamdhip64" in line}
    assert len(paths) == 1
    L = ctypes.CDLL(paths.pop())

    class Runtime:
        def __getattr__(self, name):
            def call(*args):
                assert getattr(L, name)(*args) == 0, name
            return call

        def stream(self):
            s = ctypes.c_void_p()
            self.hipStreamCreateWithFlags(ctypes.byref(s), 1)  # does not wait for the default stream
            return s

        def capture(self, s, program):
            graph, run = ctypes.c_void_p(), ctypes.c_void_p()
            self.hipStreamBeginCapture(s, 1)  # this thread's calls
            program(s)
            self.hipStreamEndCapture(s, ctypes.byref(graph))
            self.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
            return run

    return Runtime()


def f32(rng, *shape):
    return rng.normal(size=shape).astype(np.float32)


def upload(capi, buffer, array):
    array = np.ascontiguousarray(array)
    capi.check(capi.lib().tcx_hip_memcpy_h2d(buffer.buffer.ptr, array.ctypes.data, array.nbytes, capi.stream()))


class Rows:
    """8-bit rows in device memory, with marked words before and behind them."""

    MARK = 0x5A5A5A5A

    def __init__(self, capi, rows, features, x=None):
        self.capi, self.rows, self.features = capi, rows, features
        code_words, scale_words = capi.block8_words(features)
        self.shapes = (rows, code_words), (rows, scale_words)
        self.held = [capi.DeviceArray.from_numpy(np.full(64 + a * b + 64, self.MARK, np.int32)) for a, b in self.shapes]
        self.codes, self.scales = (h.ptr + 256 for h in self.held)
        if x is not None:
            dx = capi.DeviceArray.from_numpy(x)
            capi.quantise8(dx.ptr, self.codes, self.scales, rows, features)
            capi.synchronize()

    def words(self):
        out = []
        for held, shape in zip(self.held, self.shapes):
            w = held.numpy()
            assert (w[:64] == self.MARK).all() and (w[-64:] == self.MARK).all(), "words outside the rows were written"
            out.append(w[64:-64].reshape(shape))
        return out

    def values(self):
        return cases.values(*self.words())


class Floats:
    """Float32 rows `stride` apart that begin `shift` floats into their memory, 7s around them."""

    def __init__(self, capi, rows, width, stride, shift, x=None):
        self.shape, self.stride, self.shift = (rows, width), stride, shift
        host = np.full(shift + rows * stride + 32, 7, np.float32)
        if x is not None:
            host[shift:shift + rows * stride].reshape(rows, stride)[:, :width] = x
        self.held = capi.DeviceArray.from_numpy(host)
        self.ptr = self.held.ptr + 4 * shift

    def numpy(self):
        host = self.held.numpy()
        rows, width = self.shape
        body = host[self.shift:self.shift + rows * self.stride].reshape(rows, self.stride)
        assert (host[:self.shift] == 7).all() and (host[self.shift + rows * self.stride:] == 7).all()
        assert (body[:, width:] == 7).all(), "floats between the rows were written"
        return body[:, :width]


LAYOUTS = [(5, 130, 130, 0), (5, 130, 131, 1), (3, 512, 515, 3), (2, 4099, 5000, 2), (4, 1, 9, 1), (3, 127, 128, 0)]


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_rows_of_any_layout(capi, layout):
    rows, features, stride, shift = layout
    x = f32(np.random.default_rng(features), rows, features)
    source, eight, back = Floats(capi, rows, features, stride, shift, x), Rows(capi, rows, features), Floats(capi, rows, features, stride, shift)
    capi.quantise8(source.ptr, eight.codes, eight.scales, rows, features, stride)
    capi.dequantise8(eight.codes, eight.scales, back.ptr, rows, features, stride)
    capi.synchronize()
    cases.check_quantised(*eight.words(), x)
    np.testing.assert_array_equal(back.numpy(), eight.values()[:, :features])


@pytest.mark.parametrize("layout", LAYOUTS + [(2, 33001, 33004, 1), (2, 9000, 9001, 3)], ids=str)
@pytest.mark.parametrize("place", ["apart", "residual", "x"])
def test_norm_of_any_layout(capi, layout, place):
    """Rows apart from each other at any address; the sum in a place of its own, or in that
    of the residual or the input."""
    rows, features, stride, shift = layout
    rng = np.random.default_rng(features)
    x, r, w = f32(rng, rows, features), f32(rng, rows, features), f32(rng, features)
    source, other = Floats(capi, rows, features, stride, shift, x), Floats(capi, rows, features, stride + 2, shift + 1, r)
    weight, eight = Floats(capi, 1, features, features, 1, w), Rows(capi, rows, features)
    total = {"apart": Floats(capi, rows, features, features, 3), "residual": other, "x": source}[place]
    desc = capi.rmsnorm8_desc(rows, features, 1e-5, x_stride=stride, residual_stride=stride + 2, sum_stride=total.stride)
    capi.rmsnorm8(source.ptr, eight.codes, eight.scales, desc, residual=other.ptr, weight=weight.ptr, sum=total.ptr)
    capi.synchronize()
    s, y, off = cases.rmsnorm(x, r, w, 1e-5)
    np.testing.assert_array_equal(total.numpy(), s)
    cases.check_near(*eight.words(), y, off)
    # A sum without a residual is a copy; a residual's sum need not be written.
    plain, lone = Rows(capi, rows, features), Floats(capi, rows, features, features, 0)
    source = Floats(capi, rows, features, features, 0, x)
    desc = capi.rmsnorm8_desc(rows, features, 1e-5)
    capi.rmsnorm8(source.ptr, plain.codes, plain.scales, desc, sum=lone.ptr)
    capi.synchronize()
    np.testing.assert_array_equal(lone.numpy(), x)
    other = Floats(capi, rows, features, features, 0, r)
    again = Rows(capi, rows, features)
    capi.rmsnorm8(source.ptr, again.codes, again.scales, desc, residual=other.ptr, weight=weight.ptr)
    capi.synchronize()
    np.testing.assert_array_equal(other.numpy(), r)
    for a, b in zip(again.words(), eight.words()):
        np.testing.assert_array_equal(a, b)


# rows, outputs, features: with the workspaces that these ask for and without
SPLIT = [(1, 64, 8192), (1, 4096, 4096), (5, 300, 16384), (16, 128, 11264), (20, 257, 9000), (32, 4096, 4096), (60, 500, 5000), (64, 64, 16384),
         (128, 256, 8192), (130, 700, 4000), (300, 1100, 1000), (256, 512, 4096), (512, 1024, 2048)]


@pytest.mark.parametrize("shape", SPLIT, ids=str)
def test_linear_with_and_without_workspace(capi, shape):
    """Results into rows apart from each other; the same call twice gives the same bits."""
    rows, outputs, features = shape
    rng = np.random.default_rng(sum(shape))
    x, w = Rows(capi, rows, features, f32(rng, rows, features)), Rows(capi, outputs, features, f32(rng, outputs, features))
    expected, off = cases.product(x.values(), w.values())
    stride = outputs + 3
    desc = capi.linear8_desc(rows, features, outputs, out_stride=stride)
    for space in {capi.linear8_workspace(desc), None, "half"}:
        if space == "half":
            full = capi.linear8_workspace_bytes(desc)
            space = capi.DeviceBuffer(full // 2 // 16 * 16) if full >= 64 else None
        seen = []
        for _ in range(2):
            out = Floats(capi, rows, outputs, stride, 1)
            if space is not None:
                capi.check(capi.lib().tcx_hip_fill(0, space.address, space.nbytes // 4, ctypes.c_double(float("nan")), capi.stream()))
            capi.linear8(x.codes, x.scales, w.codes, w.scales, out.ptr, desc, workspace=space)
            capi.synchronize()
            seen.append(out.numpy().copy())
        error = np.abs(seen[0] - expected)
        assert (error <= off).all(), f"off by up to {(error / off).max():.3g} of the bound"
        np.testing.assert_array_equal(seen[0], seen[1])


@pytest.mark.parametrize("shape", [(1, 200, 4096), (16, 1000, 2048), (40, 300, 1000), (200, 500, 700), (300, 1300, 512), (100, 5000, 700)], ids=str)
def test_gated_surroundings(capi, shape):
    """Nothing outside the rows is written; the same call twice gives the same bits, whatever
    the workspace held."""
    rows, outputs, features = shape
    rng = np.random.default_rng(sum(shape))
    x, w = Rows(capi, rows, features, f32(rng, rows, features)), Rows(capi, 2 * outputs, features, f32(rng, 2 * outputs, features) * np.float32(0.05))
    desc = capi.linear8_desc(rows, features, outputs, activation="silu")
    space, seen = capi.linear8_workspace(desc, gated=True), []
    for fill in (float("nan"), 1e30):
        out = Rows(capi, rows, outputs)
        if space is not None:
            capi.check(capi.lib().tcx_hip_fill(0, space.address, space.nbytes // 4, ctypes.c_double(fill), capi.stream()))
        capi.gated_linear8(x.codes, x.scales, w.codes, w.scales, out.codes, out.scales, desc, workspace=space)
        capi.synchronize()
        seen.append(out.words())
    gate, gate_off = cases.product(x.values(), w.values()[:outputs], None, "silu")
    up, up_off = cases.product(x.values(), w.values()[outputs:])
    off = gate_off * (np.abs(up) + up_off) + np.abs(gate) * up_off + cases.EPS * np.abs(gate * up)
    cases.check_near(*seen[0], gate * up, off)
    for a, b in zip(*seen):
        np.testing.assert_array_equal(a, b)


class Layer:
    """The products' half of a layer on its own buffers and workspaces."""

    def __init__(self, capi, seed, rows, width=1024, inner=900):
        self.capi, self.seed, self.sizes = capi, seed, (rows, width, inner)
        rng = np.random.default_rng(seed)
        self.first = Rows(capi, 2 * inner, width, (f32(rng, 2 * inner, width) * 0.03).astype(np.float32))
        self.second = Rows(capi, width, inner, (f32(rng, width, inner) * 0.03).astype(np.float32))
        A = capi.DeviceArray
        self.x, self.residual, self.weight, self.out, self.read = A((rows, width)), A((rows, width)), A((width,)), A((rows, width)), A((rows, width))
        self.normed, self.gated, self.last = Rows(capi, rows, width), Rows(capi, rows, inner), Rows(capi, rows, width)
        self.norm = capi.rmsnorm8_desc(rows, width, 1e-5)
        self.up, self.down = capi.linear8_desc(rows, width, inner, activation="silu"), capi.linear8_desc(rows, inner, width)
        self.spaces = [capi.linear8_workspace(self.up, gated=True), capi.linear8_workspace(self.down)]
        upload(capi, self.weight, 1 + 0.1 * f32(rng, width))

    def refill(self, turn):
        rng = np.random.default_rng(1000 * self.seed + turn)
        rows, width, _ = self.sizes
        upload(self.capi, self.x, f32(rng, rows, width))
        upload(self.capi, self.residual, f32(rng, rows, width))
        upload(self.capi, self.out, np.zeros((rows, width), np.float32))
        self.capi.synchronize()

    def run(self, s):
        capi, (rows, width, inner) = self.capi, self.sizes
        capi.rmsnorm8(self.x.ptr, self.normed.codes, self.normed.scales, self.norm, residual=self.residual.ptr, weight=self.weight.ptr,
                      sum=self.residual.ptr, s=s)
        capi.gated_linear8(self.normed.codes, self.normed.scales, self.first.codes, self.first.scales, self.gated.codes,
                           self.gated.scales, self.up, workspace=self.spaces[0], s=s)
        capi.linear8(self.gated.codes, self.gated.scales, self.second.codes, self.second.scales, self.out.ptr, self.down,
                     workspace=self.spaces[1], s=s)
        capi.quantise8(self.out.ptr, self.last.codes, self.last.scales, rows, width, s=s)
        capi.dequantise8(self.last.codes, self.last.scales, self.read.ptr, rows, width, s=s)

    def results(self):
        return [self.residual.numpy(), *self.normed.words(), *self.gated.words(), self.out.numpy(), *self.last.words(), self.read.numpy()]


def same(got, expected):
    for x, y in zip(got, expected, strict=True):
        np.testing.assert_array_equal(x.view(np.int32), y.view(np.int32))


@pytest.mark.parametrize("rows", [1, 24, 300])
def test_captured_and_replayed(capi, runtime, rows):
    """Replays with new values between them, the program's own copies and waits among them,
    give what the calls give."""
    layer, s, expected = Layer(capi, 1, rows), runtime.stream(), []
    for turn in range(4):
        layer.refill(turn)
        layer.run(s)
        runtime.hipStreamSynchronize(s)
        expected.append(layer.results())
    again = Layer(capi, 1, rows)
    again.refill(0)
    graph = runtime.capture(s, again.run)
    assert not again.out.numpy().any()  # nothing ran yet
    for turn in range(4):
        again.refill(turn)
        runtime.hipGraphLaunch(graph, s)
        runtime.hipStreamSynchronize(s)
        same(again.results(), expected[turn])


def test_two_graphs_on_two_streams(capi, runtime):
    """Graphs with workspaces of their own run side by side."""
    layers, streams = [Layer(capi, 2, 8), Layer(capi, 3, 200, 768, 700)], [runtime.stream(), runtime.stream()]
    graphs = [runtime.capture(s, layer.run) for layer, s in zip(layers, streams)]
    for turn in range(3):
        expected = []
        for layer, s in zip(layers, streams):
            layer.refill(turn)
            layer.run(s)
            runtime.hipStreamSynchronize(s)
            expected.append(layer.results())
        for layer in layers:
            layer.refill(turn)
        for graph, s in zip(graphs, streams):
            runtime.hipGraphLaunch(graph, s)
        for s in streams:
            runtime.hipStreamSynchronize(s)
        for layer, want in zip(layers, expected):
            same(layer.results(), want)


def test_two_threads(capi, runtime):
    """Calls of two threads, each on its own stream and buffers."""
    layers, streams = [Layer(capi, 4, 5), Layer(capi, 5, 150, 512, 600)], [runtime.stream(), runtime.stream()]
    expected, failures = [], []
    for layer, s in zip(layers, streams):
        layer.refill(0)
        layer.run(s)
        runtime.hipStreamSynchronize(s)
        expected.append(layer.results())
        layer.refill(0)

    def work(layer, s):
        try:
            for _ in range(30):
                layer.run(s)
                runtime.hipStreamSynchronize(s)
        except BaseException as e:  # noqa: BLE001 - reported by the test's thread
            failures.append(e)

    threads = [threading.Thread(target=work, args=pair) for pair in zip(layers, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for layer, s, want in zip(layers, streams, expected):
        layer.refill(0)
        layer.run(s)
        runtime.hipStreamSynchronize(s)
        same(layer.results(), want)


def test_two_threads_results(capi, runtime):
    """Calls of two threads at the same time, each on its own stream, buffers and workspaces:
    what every turn of each gives is what its calls give alone."""
    layers, streams = [Layer(capi, 6, 7), Layer(capi, 7, 130, 512, 600)], [runtime.stream(), runtime.stream()]
    turns, failures, start = 4, [], threading.Barrier(2)

    def results(layer, s, turn):
        layer.refill(turn)
        for _ in range(8):  # the norm's sum goes to its residual: each time another one
            layer.run(s)
        runtime.hipStreamSynchronize(s)
        return layer.results()

    def work(layer, s, alone):
        try:
            start.wait(60)
            for turn in range(3 * turns):
                same(results(layer, s, turn % turns), alone[turn % turns])
        except BaseException as e:  # noqa: BLE001 - reported by the test's thread
            failures.append(e)

    expected = [[results(layer, s, turn) for turn in range(turns)] for layer, s in zip(layers, streams)]
    threads = [threading.Thread(target=work, args=args) for args in zip(layers, streams, expected)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


def test_past_32_bit_offsets(capi):
    """Rows 5 GB into their matrices: codes, float32 rows and results."""
    rng = np.random.default_rng(41)
    features, rows, keep = 2048, 2_700_000, 5  # 5.5 GB of codes
    big = capi.DeviceBuffer(rows * features)
    exponents = capi.DeviceBuffer(rows * 16)
    x, w = f32(rng, keep, features), f32(rng, 30, features)
    first = rows - keep
    dx = capi.DeviceArray.from_numpy(x)
    capi.quantise8(dx.ptr, big.address + first * features, exponents.address + first * 16, keep, features)
    weights = Rows(capi, 30, features, w)
    # As weights of which only the last tile's rows are of interest, results 2_700_000 a row.
    out = capi.DeviceBuffer(4 * rows * 30)
    desc = capi.linear8_desc(30, features, rows)
    capi.linear8(weights.codes, weights.scales, big.address, exponents.address, out.address, desc, workspace=capi.linear8_workspace(desc))
    # As activations.
    tall = capi.DeviceBuffer(4 * rows * 30)
    desc = capi.linear8_desc(rows, features, 30)
    capi.linear8(big.address, exponents.address, weights.codes, weights.scales, tall.address, desc, workspace=capi.linear8_workspace(desc))
    read = capi.DeviceArray((keep, features))
    capi.dequantise8(big.address + first * features, exponents.address + first * 16, read.ptr, keep, features)
    capi.synchronize()
    back = read.numpy()
    units, e = cases.quantise(x)
    np.testing.assert_array_equal(back, (units * 2.0 ** e[..., None]).reshape(keep, features))
    expected, off = cases.product(back.astype(float), weights.values())
    for r in (0, 17, 29):
        row = np.empty(keep, np.float32)
        capi.check(capi.lib().tcx_hip_memcpy_d2h(row.ctypes.data, out.address + 4 * (r * rows + first), row.nbytes, capi.stream()))
        assert (np.abs(row - expected[:, r]) <= off[:, r]).all()
    got = np.empty((keep, 30), np.float32)
    capi.check(capi.lib().tcx_hip_memcpy_d2h(got.ctypes.data, tall.address + 4 * 30 * first, got.nbytes, capi.stream()))
    assert (np.abs(got - expected) <= off).all()
