"""The decode step with weights in captured graphs: two graphs with workspaces of their own, replayed in turn with
eager calls between, every replay checked; each of its kernels (a wave or a workgroup a row-head, chunks of keys, tiles)."""

import numpy as np
import pytest

from tests import attention_ref as ref
from tests.test_gpu_tree_cache import RULE, TABLE, Gpu, caches
from tests.test_gpu_tree_cache_streams import Stream, ok, runtime

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


class Step:
    def __init__(self, gpu, seed, b, h, hd, cap, table):
        self.gpu, self.dims, self.table = gpu, (b, 1, h, hd, cap), table
        r = np.random.default_rng(seed)
        self.q = r.integers(-128, 128, (b, 1, h, hd)).astype(np.int8)
        self.k, self.v = caches(r, b, h, cap, hd)
        self.ctx = np.resize(np.array([cap, 1, cap // 2, 0], np.uint32), b)
        self.acc, self.out = np.zeros((b, h, cap), np.uint64), np.zeros_like(self.q)
        self.need = max(256, gpu.hip.attend_rows_workspace(*self.dims))
        self.d = [gpu(x) for x in (self.q, self.k, self.v, self.ctx)] + [None, gpu(self.acc)]
        self.d_out, self.rule, self.space = gpu(self.out), gpu.rule(RULE, table), gpu(np.zeros(self.need, np.uint8))

    def run(self, stream):
        self.gpu.hip.attend_mass(self.gpu.dev, *self.d, self.dims, self.rule, self.d_out, self.space, self.need, stream.h)

    def host(self):
        ref.mass(self.q, self.k, self.v, self.ctx, None, self.acc, RULE, self.table, self.out)

    def check(self):
        assert np.array_equal(self.gpu.back(self.d_out, self.out), self.out)
        assert np.array_equal(self.gpu.back(self.d[5], self.acc), self.acc)


@pytest.mark.parametrize("b,h,hd,cap,table", [(4, 3, 64, 200, TABLE), (4, 3, 64, 900, TABLE), (4, 2, 128, 700, TABLE),
                                              (4, 2, 64, 2100, np.resize(TABLE, 20_000)), (4, 2, 80, 600, TABLE),
                                              (4, 2, 64, 2600, TABLE), (4, 2, 20, 90, TABLE)])
def test_replayed_decode_steps(gpu, b, h, hd, cap, table):
    print(f"decode step {b}x{h}x{hd} cap {cap}", flush=True)
    rt = runtime()
    one, two, other = [Step(gpu, seed, b, h, hd, cap, table) for seed in (1, 2, 3)]
    stream = Stream(rt)
    other.run(stream)
    other.host()
    stream.sync()
    other.check()
    graphs = [(s, stream.capture(lambda: s.run(stream))) for s in (one, two)]
    for _ in range(3):
        for s, g in graphs:
            ok(rt.hipGraphLaunch(g, stream.h))
            s.host()
        other.run(stream)
        other.host()
        stream.sync()
        for s in (one, two, other):
            s.check()
    for _, g in graphs:
        ok(rt.hipGraphExecDestroy(g))
