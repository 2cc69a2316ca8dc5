"""The tree and cache operators on streams of the caller's and in captured graphs: two replayed graphs with
workspaces of their own, eager work between the replays, and every replay checked; calls on two streams at
once; calls whose workspace is too small."""

import ctypes as C

import numpy as np
import pytest

from tests import attention_ref as ref
from tests.test_gpu_tree_cache import RULE, TABLE, Gpu, caches, masks

pytestmark = pytest.mark.gpu

DEFAULT_STREAM_MODE = 2  # hipStreamCaptureModeRelaxed


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


def runtime():
    """The HIP runtime that the library has loaded."""
    for line in open("/proc/self/maps"):
        if "libamdhip64" in line:
            return C.CDLL(line.split()[-1])
    raise RuntimeError("no HIP runtime is loaded")


def ok(status):
    assert status == 0


class Stream:
    def __init__(self, rt):
        self.rt, self.h = rt, C.c_void_p()
        ok(rt.hipStreamCreate(C.byref(self.h)))

    def sync(self):
        ok(self.rt.hipStreamSynchronize(self.h))

    def capture(self, fn):
        graph, run = C.c_void_p(), C.c_void_p()
        ok(self.rt.hipStreamBeginCapture(self.h, DEFAULT_STREAM_MODE))
        fn()
        ok(self.rt.hipStreamEndCapture(self.h, C.byref(graph)))
        ok(self.rt.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)))
        ok(self.rt.hipGraphDestroy(graph))
        return run


class Step:
    """One serving step of all four operators on device buffers: attention with weights, a tree, its
    accepted path and the cut to the budget; `host` runs the same on the host's copies."""

    def __init__(self, gpu, seed, b, t, h, hd, cap, budget):
        self.gpu, self.dims = gpu, (b, t, h, hd, cap)
        self.budget, self.recent = budget, budget // 4
        r = np.random.default_rng(seed)
        self.q = r.integers(-128, 128, (b, t, h, hd)).astype(np.int8)
        self.k, self.v = caches(r, b, h, cap, hd)
        self.ctx = np.full(b, cap - t, np.uint32)
        self.keys = self.ctx + np.uint32(t)
        self.mask = masks(gpu, r, b, t)
        self.acc = np.zeros((1, b, h, cap), np.uint64)
        self.path = np.stack([np.sort(r.permutation(t)) for _ in range(b)]).astype(np.uint32)
        self.path[:, :3] = [[0, 2, 5]] * b
        self.accepted = np.full(b, 3, np.uint32)
        self.tree, self.mass = np.zeros_like(self.q), np.zeros_like(self.q)
        self.after, self.cut = np.zeros(b, np.uint32), np.zeros(b, np.uint32)
        names = ("q", "k", "v", "ctx", "keys", "mask", "acc", "path", "accepted", "tree", "mass", "after", "cut")
        self.d = {n: gpu(getattr(self, n)) for n in names}
        self.rule = gpu.rule(RULE, TABLE)
        self.need = gpu.hip.attend_rows_workspace(*self.dims)
        self.space = gpu(np.zeros(max(self.need, 256), np.uint8))

    def run(self, stream):
        g, d, hip = self.gpu, self.d, self.gpu.hip
        b, t, h, hd, cap = self.dims
        w = (self.space, max(self.need, 256), stream.h)
        hip.attend_mass(g.dev, d["q"], d["k"], d["v"], d["keys"], None, d["acc"], self.dims, self.rule, d["mass"], *w)
        hip.attend_tree(g.dev, d["q"], d["k"], d["v"], d["ctx"], None, d["mask"], self.dims, self.rule, d["tree"], *w)
        hip.cache_commit(g.dev, [d["k"]], [d["v"]], d["ctx"], d["path"], d["accepted"], self.dims, d["after"], stream.h)
        hip.cache_evict(g.dev, [d["k"]], [d["v"]], d["acc"], d["after"], (b, h, hd, cap), self.budget, self.recent,
                        d["acc"], d["cut"], None, stream.h)

    def host(self):
        ref.mass(self.q, self.k, self.v, self.keys, None, self.acc[0], RULE, TABLE, self.mass)
        ref.tree(self.q, self.k, self.v, self.ctx, None, self.mask, RULE, TABLE, self.tree)
        ref.commit([self.k], [self.v], self.ctx, self.path, self.accepted, self.after)
        ref.evict([self.k], [self.v], self.acc, self.after, self.budget, self.recent, self.acc, self.cut, None)

    def check(self):
        for n in ("mass", "tree", "after", "cut", "acc", "k", "v"):
            assert np.array_equal(self.gpu.back(self.d[n], getattr(self, n)), getattr(self, n)), n


# one launch, the long form with its workspace, the row form, the decode step
SHAPES = [(2, 8, 2, 64, 300, 200), (2, 20, 3, 64, 4300, 1000), (2, 9, 2, 20, 90, 60), (3, 6, 1, 128, 2200, 500)]


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
        other.run(stream)  # eager work between the replays
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
    for _ in range(4):
        for s, st in zip(steps, streams):
            s.run(st)
    for s, st in zip(steps, streams):
        st.sync()
        for _ in range(4):
            s.host()
        s.check()


def test_a_workspace_that_is_too_small_is_refused(gpu):
    s = Step(gpu, 9, *SHAPES[1])
    assert s.need > 0
    hip, d = gpu.hip, s.d
    for space, size in ((s.space, s.need - 1), (s.space.value + 16, s.need)):
        with pytest.raises(hip.HipError) as e:
            hip.attend_tree(gpu.dev, d["q"], d["k"], d["v"], d["ctx"], None, d["mask"], s.dims, s.rule, d["tree"], space, size)
        assert e.value.status == hip.HS_INVALID_ARGUMENT
    hip.attend_tree(gpu.dev, d["q"], d["k"], d["v"], d["ctx"], None, d["mask"], s.dims, s.rule, d["tree"])  # its own
    ref.tree(s.q, s.k, s.v, s.ctx, None, s.mask, RULE, TABLE, s.tree)
    assert np.array_equal(gpu.back(d["tree"], s.tree), s.tree)


def test_a_captured_call_without_a_workspace_is_refused(gpu):
    rt = runtime()
    s, stream = Step(gpu, 11, *SHAPES[1]), Stream(rt)
    s.run(stream)
    s.host()
    stream.sync()
    s.check()
    hip, d = gpu.hip, s.d
    refused = []

    def fn():
        for call, third in ((hip.attend_tree, d["mask"]), (hip.attend_mass, d["acc"])):
            try:
                call(gpu.dev, d["q"], d["k"], d["v"], d["keys"], None, third, s.dims, s.rule, d["tree"], None, 0, stream.h)
            except hip.HipError as e:
                refused.append(e.status)
        s.run(stream)  # the capture goes on

    run = stream.capture(fn)
    assert refused == [hip.HS_INVALID_ARGUMENT] * 2
    for _ in range(2):
        ok(rt.hipGraphLaunch(run, stream.h))
        s.host()
        stream.sync()
        s.check()
    ok(rt.hipGraphExecDestroy(run))
