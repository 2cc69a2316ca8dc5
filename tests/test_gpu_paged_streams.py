"""Paged caches and scores on streams of the caller's and in captured graphs: replayed graphs that append and attend with
counts that advance on the device and workspaces of their own, eager work between the replays, every replay checked; two
streams at once; a pool that two streams share; workspaces that are too small; calls from two threads."""

import threading

import numpy as np
import pytest

from tests import paged_ref as ref
from tests.test_gpu_paged import RULE, check_pool, device_cache, new_rows, tables
from tests.test_gpu_scores import WEIGHTS
from tests.test_gpu_tree_cache import TABLE, Gpu
from tests.test_gpu_tree_cache_streams import Stream, ok, runtime

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


class Step:
    """Two tokens (or chunks) of a layer on device buffers, whose counts go from one buffer to the other and back, and the
    scores of some logits; `host` runs the same on the host's copies."""

    def __init__(self, gpu, seed, b, t, heads, kvh, hd, page, width, start, table=TABLE):
        self.gpu, self.table_exp = gpu, table
        r = np.random.default_rng(seed)
        self.pool = ref.Pool(r, b * width + 1, kvh, page, hd, 64)
        self.cache, self.table = device_cache(gpu, self.pool), tables(r, b, width, b * width + 1)
        self.dims, self.keys = (b, t, heads, width), width * page
        self.q = r.integers(-128, 128, (b, t, heads, hd)).astype(np.int8)
        self.k, self.v = new_rows(r, b, t, kvh, hd, 16)
        self.counts = [np.full(b, start, np.uint32), np.zeros(b, np.uint32)]
        self.out = np.zeros_like(self.q)
        self.logits = np.rint(r.standard_normal((b, 3000)) * 700).astype(np.int32)
        self.top, self.logprob = np.zeros((b, 5), np.uint32), np.zeros((b, 5), np.float32)
        self.d = {n: gpu(getattr(self, n)) for n in ("q", "k", "v", "table", "out", "logits", "top", "logprob")}
        self.d_counts, self.weights, self.rule = [gpu(x) for x in self.counts], gpu(WEIGHTS), gpu.rule(RULE, table)
        self.need = gpu.hip.attend_paged_workspace(b, t, heads, kvh, hd, self.keys)
        self.space = gpu(np.zeros(max(self.need, 256), np.uint8))

    def run(self, stream, workspace=True):
        g, d, hip = self.gpu, self.d, self.gpu.hip
        b, t, heads, width = self.dims
        for i in range(2):
            now, after = self.d_counts[i], self.d_counts[1 - i]
            hip.pages_append(g.dev, self.cache, d["k"], d["v"], d["table"], now, None, (b, t, width), 20, after, bits=16,
                             stream=stream.h)
            w = dict(workspace=self.space, workspace_bytes=max(self.need, 256)) if workspace else {}
            hip.attend_paged(g.dev, self.cache, d["q"], d["table"], after, None, (b, t, heads, width, self.keys), self.rule,
                             d["out"], stream=stream.h, **w)
        hip.score_tokens(g.dev, d["logits"], None, self.weights, (b, 3000, len(WEIGHTS)), 5, None, None, None, d["top"],
                         d["logprob"], bits=32, stream=stream.h)

    def host(self):
        for i in range(2):
            after = np.zeros_like(self.counts[0])
            ref.append(self.pool, self.k, self.v, self.table, self.counts[i], None, 20, after)
            self.counts[1 - i] = after
            ref.attend(self.pool, self.q, self.table, after, None, self.keys, RULE, self.table_exp, self.out)
        self.top = ref.scores(self.logits, WEIGHTS, None, 5)[3]

    def check(self):
        check_pool(self.gpu, self.cache, self.pool)
        for n in ("out", "top"):
            assert np.array_equal(self.gpu.back(self.d[n], getattr(self, n)), getattr(self, n)), n
        for d, x in zip(self.d_counts, self.counts):
            assert np.array_equal(self.gpu.back(d, x), x)


# one launch of 4, 16 and 8 rows, launches that keep the scores (1 row past 8,192 keys), three walks, 8 rows past 4,096 keys
SHAPES = [(2, 1, 3, 3, 64, 16, 20, 300), (2, 7, 4, 2, 64, 32, 16, 300), (2, 1, 16, 2, 128, 64, 40, 2200),
          (1, 1, 2, 2, 64, 128, 66, 8300), (2, 20, 3, 3, 64, 64, 44, 2500),
          (2, 1, 16, 2, 128, 64, 70, 4200)]


@pytest.mark.parametrize("shape", SHAPES)
def test_replayed_graphs(gpu, shape):
    rt = runtime()
    one, two, stream = Step(gpu, 1, *shape), Step(gpu, 2, *shape), Stream(rt)
    other = Step(gpu, 3, *shape)
    other.run(stream)  # eager first: kernels loaded, attributes set
    other.host()
    stream.sync()
    other.check()
    graphs = [(s, stream.capture(lambda: s.run(stream))) for s in (one, two)]
    for _ in range(3):
        for s, g in graphs:
            ok(rt.hipGraphLaunch(g, stream.h))
            s.host()
        other.run(stream, workspace=False)  # eager work between the replays, in memory of the device's pool
        other.host()
        stream.sync()
        for s in (one, two, other):
            s.check()
    for _, g in graphs:
        ok(rt.hipGraphExecDestroy(g))


@pytest.mark.parametrize("shape", SHAPES)
def test_two_streams_at_once(gpu, shape):
    rt = runtime()
    steps, streams = [Step(gpu, 5 + i, *shape) for i in range(2)], [Stream(rt), Stream(rt)]
    for i in range(4):
        for s, st in zip(steps, streams):
            s.run(st, workspace=i % 2 == 0)
    for s, st in zip(steps, streams):
        st.sync()
        for _ in range(4):
            s.host()
        s.check()


def test_two_threads(gpu):
    """Calls from two host threads, each on a stream of its own."""
    rt = runtime()
    steps = [Step(gpu, 20 + i, *SHAPES[2 * i]) for i in range(2)]
    failed = []

    def work(s):
        try:
            st = Stream(rt)
            for _ in range(6):
                s.run(st, workspace=False)
            st.sync()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in steps]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for s in steps:
        for _ in range(6):
            s.host()
        s.check()


def test_streams_that_share_pages(gpu):
    """A prompt's pages that two streams read, each with pages of its own behind them."""
    r = np.random.default_rng(7)
    pool = ref.Pool(r, 8, 2, 16, 64, 64)
    cache, table = device_cache(gpu, pool), np.array([[5, 1, 0, 2], [5, 1, 3, 4]], np.uint32)
    ctx, q = np.array([40, 37], np.uint32), r.integers(-128, 128, (2, 3, 2, 64)).astype(np.int8)
    k, v = new_rows(r, 2, 3, 2, 64, 16)
    after, out = gpu(np.zeros(2, np.uint32)), np.zeros_like(q)
    d_table, d_out = gpu(table), gpu(out)
    gpu.hip.pages_append(gpu.dev, cache, gpu(k), gpu(v), d_table, gpu(ctx), None, (2, 3, 4), 20, after, bits=16)
    gpu.hip.attend_paged(gpu.dev, cache, gpu(q), d_table, after, None, (2, 3, 2, 4, 64), gpu.rule(RULE, TABLE), d_out)
    counts = np.zeros(2, np.uint32)
    ref.append(pool, k, v, table, ctx, None, 20, counts)
    check_pool(gpu, cache, pool)
    assert np.array_equal(gpu.back(d_out, out), ref.attend(pool, q, table, counts, None, 64, RULE, TABLE, out))


def test_workspaces(gpu):
    """One that is too small or not aligned is refused, and so is a captured call without one."""
    rt, hip = runtime(), gpu.hip
    s, stream = Step(gpu, 9, *SHAPES[3]), Stream(rt)
    b, t, heads, width = s.dims
    assert s.need > 0
    call = lambda **kw: hip.attend_paged(gpu.dev, s.cache, s.d["q"], s.d["table"], s.d_counts[0], None,  # noqa: E731
                                         (b, t, heads, width, s.keys), s.rule, s.d["out"], **kw)
    for space, size in ((s.space, s.need - 1), (s.space.value + 16, s.need)):
        with pytest.raises(hip.HipError) as e:
            call(workspace=space, workspace_bytes=size)
        assert e.value.status == hip.HS_INVALID_ARGUMENT
    s.run(stream)
    s.host()
    stream.sync()
    s.check()
    refused = []

    def fn():
        try:
            call(stream=stream.h)
        except hip.HipError as e:
            refused.append(e.status)
        s.run(stream)  # the capture goes on

    run = stream.capture(fn)
    assert refused == [hip.HS_INVALID_ARGUMENT]
    for _ in range(2):
        ok(rt.hipGraphLaunch(run, stream.h))
        s.host()
        stream.sync()
        s.check()
    ok(rt.hipGraphExecDestroy(run))
