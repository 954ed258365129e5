"""GPU tests of how the decoding operators are called: every form of the windowed
attention, captured graphs, several streams and threads, addresses of any
alignment, tensors past 32-bit offsets, and candidates that all tie.

Results of the same call are compared bit for bit; those against the plain
forms with the tolerances of decoding_cases."""

from __future__ import annotations

import ctypes
import threading

import numpy as np
import pytest

import decoding_cases as cases
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


class Loop:
    """One step of a decoding loop on its own buffers and workspaces."""

    def __init__(self, capi, seed, batch=2, beams=3, heads=8, kv=2, d=128, cols=1500, vocabulary=9000, prompt=0):
        self.capi, self.seed = capi, seed
        rows = self.rows = batch * beams
        self.sizes = batch, beams, heads, kv, d, cols, vocabulary
        A = capi.DeviceArray
        self.q, self.k, self.v = A((rows, heads, 1, d)), A((rows, kv, cols, d)), A((rows, kv, cols, d))
        words = d // 8 + d // 32
        self.caches = [A((rows, kv, cols, words), np.int32) for _ in range(4)]
        self.positions, self.lengths = A((rows,), np.int32), A((rows,), np.int32)
        self.logits, self.scores = A((batch, beams, vocabulary)), A((batch, beams))
        self.out = [A((rows, heads, 1, d)), A((rows, heads, 1, d)), A((batch, beams)), A((batch, beams), np.int32),
                    A((batch, beams), np.int32)]
        self.new_k, self.new_v = A((rows, kv, 1, d)), A((rows, kv, 1, d))
        desc = lambda **more: capi.window_attention_desc(rows, heads, kv, 1, cols, d, lengths=self.lengths.ptr, **more)
        self.window, self.cached = desc(window=1100, sinks=3), desc()
        self.store = capi.cache4_store_desc(rows, kv, 1, cols, d)
        self.spaces = [capi.window_attention_workspace(self.window), capi.window_attention_workspace(self.cached, cache=True),
                       capi.beam_select_workspace(batch, beams, vocabulary, beams)]
        assert all(s is not None for s in self.spaces)  # splits and their join are part of it
        self.plan = capi.beam_reorder_plan([c.ptr for c in self.caches[:2]], [c.ptr for c in self.caches[2:]],
                                           [kv * cols * words * 4] * 2)
        rng = np.random.default_rng(seed)
        for buffer, kind in ((self.k, "f"), (self.v, "f")):
            upload(capi, buffer, f32(rng, *buffer.shape))
        for cache, x in zip(self.caches, (self.k, self.v)):
            upload(capi, cache, cases.cache_rows(x.numpy()))

    def refill(self, turn):
        """New values for the inputs, from the host, on the library's stream."""
        batch, beams, heads, kv, d, cols, vocabulary = self.sizes
        rng = np.random.default_rng(1000 * self.seed + turn)
        upload(self.capi, self.q, f32(rng, *self.q.shape))
        upload(self.capi, self.new_k, f32(rng, *self.new_k.shape))
        upload(self.capi, self.new_v, f32(rng, *self.new_v.shape))
        upload(self.capi, self.logits, f32(rng, *self.logits.shape))
        upload(self.capi, self.scores, f32(rng, *self.scores.shape))
        n = rng.integers(1, cols, self.rows).astype(np.int32)
        upload(self.capi, self.positions, n - 1)
        upload(self.capi, self.lengths, n)
        for out in self.out:
            upload(self.capi, out, np.zeros(out.shape, out.dtype))
        self.capi.synchronize()

    def run(self, s):
        capi = self.capi
        batch, beams, heads, kv, d, cols, vocabulary = self.sizes
        a = [x.ptr for x in self.out]
        capi.window_attention(self.q.ptr, self.k.ptr, self.v.ptr, a[0], self.window, workspace=self.spaces[0], s=s)
        capi.cache4_store(self.new_k.ptr, self.new_v.ptr, self.caches[0].ptr, self.caches[1].ptr, self.positions.ptr, self.store, s=s)
        capi.cache4_attention(self.q.ptr, self.caches[0].ptr, self.caches[1].ptr, a[1], self.cached, workspace=self.spaces[1], s=s)
        capi.beam_select(self.logits.ptr, self.scores.ptr, a[2], a[3], a[4], batch, beams, vocabulary, beams,
                         workspace=self.spaces[2], s=s)
        capi.beam_reorder(self.plan, a[3], batch, beams, beams, s=s)

    def results(self):
        return [x.numpy() for x in (*self.out, *self.caches)]


def same(got, expected):
    for x, y in zip(got, expected, strict=True):
        np.testing.assert_array_equal(x.view(np.int32), y.view(np.int32))


def test_a_step_captured_and_replayed(capi, runtime):
    """Replays with new values between them, the program's own copies and waits
    among them, give what the calls give."""
    loop, s = Loop(capi, 1), runtime.stream()
    expected = []
    for turn in range(4):
        loop.refill(turn)
        loop.run(s)
        runtime.hipStreamSynchronize(s)
        expected.append(loop.results())
    again = Loop(capi, 1)
    again.refill(0)
    graph = runtime.capture(s, again.run)
    same(again.results()[:2], [np.zeros_like(x) for x in expected[0][:2]])  # nothing ran yet
    for turn in range(4):
        again.refill(turn)
        runtime.hipGraphLaunch(graph, s)
        runtime.hipStreamSynchronize(s)
        same(again.results(), expected[turn])


def test_two_graphs_on_two_streams(capi, runtime):
    """Graphs with workspaces of their own run side by side."""
    loops, streams = [Loop(capi, 2), Loop(capi, 3, heads=4, d=64, cols=2100)], [runtime.stream(), runtime.stream()]
    graphs = [runtime.capture(s, loop.run) for loop, s in zip(loops, streams)]
    for turn in range(3):
        expected = []
        for loop in loops:
            loop.refill(turn)
        before = [[c.numpy() for c in loop.caches] for loop in loops]
        for loop, s in zip(loops, streams):
            loop.run(s)
            runtime.hipStreamSynchronize(s)
            expected.append(loop.results())
        for loop, caches in zip(loops, before):
            loop.refill(turn)
            for c, x in zip(loop.caches, caches):
                upload(capi, c, x)
        capi.synchronize()
        for _ in range(5):
            for graph, s in zip(graphs, streams):
                runtime.hipGraphLaunch(graph, s)
        for s in streams:
            runtime.hipStreamSynchronize(s)
        for loop, want in zip(loops, expected):
            same(loop.results(), want)


def test_two_threads(capi, runtime):
    """Calls of two threads, each on its own stream and buffers."""
    loops, streams = [Loop(capi, 4), Loop(capi, 5, heads=2, d=32, cols=2500)], [runtime.stream(), runtime.stream()]
    for loop in loops:
        loop.refill(0)
    expected, failures = [], []
    for loop, s in zip(loops, streams):
        loop.run(s)
        runtime.hipStreamSynchronize(s)
        expected.append(loop.results())

    def work(loop, s):
        try:
            for _ in range(50):
                loop.run(s)
            runtime.hipStreamSynchronize(s)
        except BaseException as e:  # noqa: BLE001 - reported by the test's thread
            failures.append(e)

    threads = [threading.Thread(target=work, args=pair) for pair in zip(loops, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for loop, want in zip(loops, expected):
        same(loop.results(), want)


# (batch, heads, kv_heads, rows, cols, features, window, sinks): more than eight rows of a
# head take matrix instructions; those with many blocks pack the keys once, in
# blocks of 64, 128 or 256 rows.
PROMPTS = [
    (2, 3, 1, 3, 700, 64, None, 0),
    (1, 1, 1, 15, 900, 128, None, 2),
    (1, 1, 1, 1030, 1030, 64, 100, 3),
    (1, 2, 1, 600, 1500, 128, None, 0),
    (43, 2, 2, 257, 300, 32, 70, 5),
    (43, 2, 2, 257, 260, 128, None, 0),
    (32, 8, 4, 130, 200, 128, 50, 70),
    (128, 1, 1, 257, 257, 80, 33, 1),
]


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("shape", PROMPTS, ids=str)
def test_prompts_of_every_form(capi, runtime, shape, whole):
    """With the workspace and without: some heads against the plain form; captured and
    replayed the same bits."""
    batch, heads, kv, rows, cols, d, window, sinks = shape
    rng = np.random.default_rng(sum(shape[:6]))
    q, k, v = f32(rng, batch, heads, rows, d), f32(rng, batch, kv, cols, d), f32(rng, batch, kv, cols, d)
    lengths = rng.integers(rows // 2, cols + 1, batch).astype(np.int32)
    lengths[0] = cols
    dq, dk, dv, dn = (capi.DeviceArray.from_numpy(x) for x in (q, k, v, lengths))
    out = capi.DeviceArray.from_numpy(np.full_like(q, 7))
    desc = capi.window_attention_desc(batch, heads, kv, rows, cols, d, window=window or 0, sinks=sinks, lengths=dn.ptr)
    ws = capi.window_attention_workspace(desc) if whole else None
    assert not whole or ws is not None
    s = runtime.stream()
    capi.synchronize()
    run = lambda on: capi.window_attention(dq.ptr, dk.ptr, dv.ptr, out.ptr, desc, workspace=ws, s=on)
    run(s)
    runtime.hipStreamSynchronize(s)
    got = out.numpy()
    for b, h in {(0, 0), (batch // 2, heads - 1), (batch - 1, 0)}:
        one = np.s_[b:b + 1, h // (heads // kv):h // (heads // kv) + 1]
        expected, bound = cases.attention(q[b:b + 1, h:h + 1], k[one], v[one], lengths[b:b + 1], window, sinks, d ** -0.5)
        off = np.abs(got[b:b + 1, h:h + 1] - expected)
        assert (off <= bound).all(), (b, h)
    graph = runtime.capture(s, run)
    for _ in range(2):
        upload(capi, out, np.zeros_like(q))
        capi.synchronize()
        runtime.hipGraphLaunch(graph, s)
        runtime.hipStreamSynchronize(s)
        same([out.numpy()], [got])


def test_past_32_bit_offsets(capi):
    """The last tokens of a cache of 120 million, and sequences 4.8 GB apart."""
    rng = np.random.default_rng(41)
    cols, d, n, words = 120_000_000, 128, 70, 20
    cache, other = capi.DeviceBuffer(cols * words * 4), capi.DeviceBuffer(cols * words * 4)
    x, q = f32(rng, 1, 1, n, d), f32(rng, 1, 4, 1, d)
    dx, dq = capi.DeviceArray.from_numpy(x), capi.DeviceArray.from_numpy(q)
    at, length = (capi.DeviceArray.from_numpy(np.array([p], np.int32)) for p in (cols - n, cols))
    out, read = capi.DeviceArray(q.shape), capi.DeviceArray((1, 1, n, d))
    capi.cache4_store(dx.ptr, dx.ptr, cache.address, other.address, at.ptr, capi.cache4_store_desc(1, 1, n, cols, d))
    capi.cache4_load(other.address, read.ptr, 1, cols, cols - n, n, d)
    desc = capi.window_attention_desc(1, 4, 1, 1, cols, d, window=n, lengths=length.ptr)
    capi.cache4_attention(dq.ptr, cache.address, other.address, out.ptr, desc)
    capi.synchronize()
    rows = cases.cache_values(cases.cache_rows(x), d)
    np.testing.assert_allclose(read.numpy(), rows, rtol=cases.EPS, atol=2.0 ** -150)
    expected, bound = cases.attention(q, rows, rows, [n], None, 0, d ** -0.5)
    assert (np.abs(out.numpy() - expected) <= bound).all()

    far = 1_200_000_000  # floats of the same memory from one sequence to the next
    for rows_of in (1, 20):
        q, k = f32(rng, 2, 2, rows_of, 64), f32(rng, 2, 1, 90, 64)
        for b in range(2):
            capi.check(capi.lib().tcx_hip_memcpy_h2d(cache.address + 4 * far * b, k[b].ctypes.data, k[b].nbytes, capi.stream()))
        dq, out = capi.DeviceArray.from_numpy(q), capi.DeviceArray(q.shape)
        desc = capi.window_attention_desc(2, 2, 1, rows_of, 90, 64, k_strides=(far, 90 * 64, 64), v_strides=(far, 90 * 64, 64))
        capi.window_attention(dq.ptr, cache.address, cache.address, out.ptr, desc)
        capi.synchronize()
        expected, bound = cases.attention(q, k, k, [90, 90], None, 0, 0.125)
        assert (np.abs(out.numpy() - expected) <= bound).all()


@pytest.mark.parametrize("offset", [1, 4, 8, 16])
def test_reorder_of_any_address(capi, offset):
    rng = np.random.default_rng(offset)
    batch, beams, count, size = 2, 3, 4, 8 * 2048 + offset % 5
    x = rng.integers(0, 256, batch * beams * size).astype(np.uint8)
    source = capi.DeviceArray.from_numpy(np.concatenate([np.zeros(offset, np.uint8), x]))
    target = capi.DeviceArray.from_numpy(np.full(batch * count * size + 2 * offset, 9, np.uint8))
    index = rng.integers(0, beams, (batch, count)).astype(np.int32)
    dn = capi.DeviceArray.from_numpy(index)
    capi.beam_reorder(capi.beam_reorder_plan([source.ptr + offset], [target.ptr + offset], [size]), dn.ptr, batch, beams, count)
    capi.synchronize()
    got = target.numpy()
    rows = (np.arange(batch)[:, None] * beams + index).reshape(-1)
    np.testing.assert_array_equal(got[offset:-offset].reshape(batch * count, size), x.reshape(batch * beams, size)[rows])
    assert (got[:offset] == 9).all() and (got[-offset:] == 9).all()


def select(capi, logits, scores, count, shift=0, finished=None, eos=0):
    batch, beams, vocabulary = logits.shape
    dx = capi.DeviceArray.from_numpy(np.concatenate([np.zeros(shift, np.float32), logits.reshape(-1)]))
    ds = capi.DeviceArray.from_numpy(scores)
    outs = [capi.DeviceArray((batch, count)), *(capi.DeviceArray((batch, count), np.int32) for _ in range(2))]
    ws = capi.beam_select_workspace(batch, beams, vocabulary, count)
    capi.beam_select(dx.ptr + 4 * shift, ds.ptr, *(o.ptr for o in outs), batch, beams, vocabulary, count, workspace=ws)
    capi.synchronize()
    return [o.numpy() for o in outs]


@pytest.mark.parametrize("shape", [(1, 4, 20000, 8), (16, 8, 70000, 16)], ids=str)
@pytest.mark.parametrize("order", ["random", "rising", "falling"])
def test_select_of_any_alignment_and_order(capi, shape, order):
    """The same logits from aligned and unaligned addresses; sorted rows, whose first
    are all in one part, or in the last."""
    batch, beams, vocabulary, count = shape
    rng = np.random.default_rng(vocabulary)
    logits, scores = 3 * f32(rng, batch, beams, vocabulary), f32(rng, batch, beams)
    if order != "random":
        logits.sort(-1)
    if order == "falling":
        logits = np.ascontiguousarray(logits[..., ::-1])
    want = cases.beam_best(logits, scores, count)
    for shift in (0, 1, 2):
        got = select(capi, logits, scores, count, shift)
        np.testing.assert_array_equal(got[1], want[1])
        np.testing.assert_array_equal(got[2], want[2])
        assert (np.abs(got[0] - want[0]) <= np.abs(want[0]) * cases.EPS + 120 * cases.EPS).all()


@pytest.mark.parametrize("value", [np.nan, -np.inf, 2.0])
@pytest.mark.parametrize("beams,vocabulary,count", [(1, 30000, 200), (8, 9001, 256), (64, 300, 256), (3, 128256, 5)])
def test_select_of_ties_alone(capi, beams, vocabulary, count, value):
    """More equal candidates than any list holds: the first tokens of the first beams."""
    logits = np.full((2, beams, vocabulary), value, np.float32)
    got = select(capi, logits, np.zeros((2, beams), np.float32), count)
    flat = np.arange(count)
    for b in range(2):
        np.testing.assert_array_equal(got[1][b], flat // vocabulary)
        np.testing.assert_array_equal(got[2][b], flat % vocabulary)
    if np.isnan(value):
        assert np.isnan(got[0]).all()
    elif np.isinf(value):
        assert np.isneginf(got[0]).all()
    else:
        assert (np.abs(got[0] + np.log(vocabulary)) <= np.log(vocabulary) * cases.EPS + 120 * cases.EPS).all()


@pytest.mark.parametrize("shape", [(1, 4, 32000, 8), (16, 8, 40000, 16), (1, 2, 2048, 3)], ids=str)
@pytest.mark.parametrize("kept", [0.3, 0.01, 0.0005])
def test_select_of_masked_logits(capi, shape, kept):
    """Most tokens at -inf, in some parts of a row all of them."""
    batch, beams, vocabulary, count = shape
    rng = np.random.default_rng(vocabulary)
    logits, scores = f32(rng, batch, beams, vocabulary), f32(rng, batch, beams)
    logits[rng.random(logits.shape) >= kept] = -np.inf
    want, got = cases.beam_best(logits, scores, count), select(capi, logits, scores, count)
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[2], want[2])
    seen = np.isfinite(want[0])
    assert np.isneginf(got[0][~seen]).all()
    assert (np.abs(got[0][seen] - want[0][seen]) <= np.abs(want[0][seen]) * cases.EPS + 120 * cases.EPS).all()


def test_select_behind_a_far_score(capi):
    """A beam at -1e30 whose scores all round to the same: the larger logits first, after
    every token of the other beam."""
    rng = np.random.default_rng(51)
    logits = f32(rng, 1, 2, 9000)
    logits[0, 0, 20:] = -np.inf
    got = select(capi, logits, np.array([[0, -1e30]], np.float32), 40)
    assert got[1][0].tolist() == [0] * 20 + [1] * 20
    np.testing.assert_array_equal(got[2][0, :20], np.argsort(-logits[0, 0, :20], kind="stable"))
    np.testing.assert_array_equal(got[2][0, 20:], np.argsort(-logits[0, 1], kind="stable")[:20])


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("vocabulary", [50, 40000])
def test_select_of_a_lost_beam(capi, vocabulary, value):
    """NaN or +inf makes its beam's candidates NaN, which come first, by their logits."""
    rng = np.random.default_rng(52)
    logits = f32(rng, 1, 3, vocabulary)
    logits[0, 1, 37] = value
    got = select(capi, logits, np.zeros((1, 3), np.float32), 5)
    assert np.isnan(got[0]).all() and got[1][0].tolist() == [1] * 5
    rest = np.where(np.arange(vocabulary) == 37, -np.inf, logits[0, 1])
    np.testing.assert_array_equal(got[2][0], [37, *np.argsort(-rest, kind="stable")[:4]])


@pytest.mark.parametrize("batch,heads,kv,rows", [(1, 2, 1, 20), (2, 4, 4, 300), (3, 8, 2, 1), (64, 8, 8, 130)])
def test_no_keys(capi, batch, heads, kv, rows):
    """Without keys every row is zeros, in each form, with the workspace that the query asks for."""
    q = capi.DeviceArray.from_numpy(np.ones((batch, heads, rows, 64), np.float32))
    out = capi.DeviceArray.from_numpy(np.full((batch, heads, rows, 64), 7, np.float32))
    desc = capi.window_attention_desc(batch, heads, kv, rows, 0, 64)
    capi.window_attention(q.ptr, None, None, out.ptr, desc, workspace=capi.window_attention_workspace(desc))
    capi.synchronize()
    assert (out.numpy() == 0).all()
    n = capi.DeviceArray.from_numpy(np.zeros(batch, np.int32))
    cache = capi.DeviceArray.from_numpy(np.full((batch, kv, 700, 10), 0x7fc07fc0, np.int32))
    out = capi.DeviceArray.from_numpy(np.full((batch, heads, rows, 64), 7, np.float32))
    desc = capi.window_attention_desc(batch, heads, kv, rows, 700, 64, lengths=n.ptr)
    ws = capi.window_attention_workspace(desc, cache=True)
    capi.cache4_attention(q.ptr, cache.ptr, cache.ptr, out.ptr, desc, workspace=ws)
    capi.synchronize()
    assert (out.numpy() == 0).all()
