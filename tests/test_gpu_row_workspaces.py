"""The row attention's calls without a workspace: many at once on several streams, whose memory comes from the
device's pool, and a device that is closed before they are done."""

import numpy as np
import pytest

from tests import attention_ref as ref
from tests.test_gpu_tree_cache import RULE, TABLE, Gpu, caches, masks
from tests.test_gpu_tree_cache_streams import Stream, runtime

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


class Job:
    """A tree or a causal chunk over caches long enough to need a workspace."""

    def __init__(self, gpu, seed, b, t, h, hd, cap, tree):
        self.gpu, self.dims, self.tree = gpu, (b, t, h, hd, cap), tree
        r = np.random.default_rng(seed)
        self.q = r.integers(-128, 128, (b, t, h, hd)).astype(np.int8)
        self.k, self.v = caches(r, b, h, cap, hd)
        self.ctx = np.full(b, cap - t if tree else cap, np.uint32)
        self.third = masks(gpu, r, b, t) if tree else np.zeros((b, h, cap), np.uint64)
        self.out = np.zeros_like(self.q)
        assert gpu.hip.attend_rows_workspace(*self.dims) > 0
        self.d = [gpu(x) for x in (self.q, self.k, self.v, self.ctx)] + [None, gpu(self.third)]
        self.d_out, self.rule = gpu(self.out), gpu.rule(RULE, TABLE)

    def run(self, dev, stream):
        fn = self.gpu.hip.attend_tree if self.tree else self.gpu.hip.attend_mass
        fn(dev, *self.d, self.dims, self.rule, self.d_out, stream=stream.h)

    def check(self, calls):
        if self.tree:
            ref.tree(self.q, self.k, self.v, self.ctx, None, self.third, RULE, TABLE, self.out)
        else:
            ref.mass(self.q, self.k, self.v, self.ctx, None, self.third, RULE, TABLE, self.out)
            self.third *= np.uint64(calls)
            assert np.array_equal(self.gpu.back(self.d[5], self.third), self.third)
        assert np.array_equal(self.gpu.back(self.d_out, self.out), self.out)


SHAPES = [(3, 20, 2, 64, 2600, True), (2, 40, 3, 64, 4200, False), (1, 5, 2, 128, 3000, True), (2, 3, 1, 256, 2500, False)]


def test_streams_share_the_pool(gpu):
    """Four streams that take and give back memory of different sizes, interleaved; synchronizations between."""
    rt = runtime()
    jobs, streams = [Job(gpu, 30 + i, *s) for i, s in enumerate(SHAPES)], [Stream(rt) for _ in SHAPES]
    calls = 0
    for turn in range(3):
        for _ in range(6):
            for job, s in zip(jobs, streams):
                job.run(gpu.dev, s)
            calls += 1
        streams[turn].sync()
    for s in streams:
        s.sync()
    for job in jobs:
        job.check(calls)


def test_a_device_closed_before_its_calls_are_done(gpu):
    """The pool goes with the device: closing waits for the calls that work in its memory."""
    rt = runtime()
    jobs, streams = [Job(gpu, 40 + i, *s) for i, s in enumerate(SHAPES)], [Stream(rt) for _ in SHAPES]
    dev = gpu.hip.HipDevice.open(0)
    for _ in range(5):
        for job, s in zip(jobs, streams):
            job.run(dev, s)
    dev.close()
    for s in streams:
        s.sync()
    for job in jobs:
        job.check(5)
