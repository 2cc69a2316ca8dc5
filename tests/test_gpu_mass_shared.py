"""Calls of attention with weights on two streams at once that add to the same accumulators: no form loses an
addition."""

import numpy as np
import pytest

from tests import attention_ref as ref
from tests.test_gpu_tree_cache import RULE, TABLE, Gpu, caches
from tests.test_gpu_tree_cache_streams import Stream, runtime

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


# one row: a wave a row-head, a workgroup a row-head, chunks of keys; several rows: tiles, ranges, the row form
@pytest.mark.parametrize("b,t,h,hd,cap,table", [
    (48, 1, 12, 64, 200, TABLE), (48, 1, 12, 64, 900, TABLE), (48, 1, 12, 32, 900, TABLE), (48, 1, 12, 128, 900, TABLE),
    (24, 1, 12, 64, 2100, np.resize(TABLE, 20_000)), (24, 3, 12, 64, 700, TABLE), (12, 3, 4, 64, 2100, TABLE),
    (24, 3, 4, 20, 200, TABLE)])
def test_two_streams_add_to_the_same_accumulators(gpu, b, t, h, hd, cap, table):
    print(f"mass {b}x{t}x{h}x{hd} cap {cap}", flush=True)
    r, rt, calls = np.random.default_rng(12), runtime(), 12
    streams = [Stream(rt), Stream(rt)]
    q = r.integers(-128, 128, (b, t, h, hd)).astype(np.int8)
    kc, vc = caches(r, 2, h, cap, hd)
    kc, vc = np.tile(kc, (b // 2, 1, 1, 1)), np.tile(vc, (b // 2, 1, 1, 1))
    q = np.tile(q[:2], (b // 2, 1, 1, 1))  # two different streams' worth, many times
    ctx = np.resize(np.array([cap, cap - 9], np.uint32), b)
    acc, out = np.zeros((b, h, cap), np.uint64), np.zeros_like(q)
    dq, dk, dv, d_ctx, d_acc, rule = gpu(q), gpu(kc), gpu(vc), gpu(ctx), gpu(acc), gpu.rule(RULE, table)
    need = gpu.hip.attend_rows_workspace(b, t, h, hd, cap)
    outs, spaces = [gpu(out), gpu(out)], [gpu(np.zeros(max(need, 256), np.uint8)) for _ in range(2)]
    for _ in range(calls):
        for s, o, w in zip(streams, outs, spaces):
            gpu.hip.attend_mass(gpu.dev, dq, dk, dv, d_ctx, None, d_acc, (b, t, h, hd, cap), rule, o, w, max(need, 256), s.h)
    for s in streams:
        s.sync()
    one = np.zeros((2, h, cap), np.uint64)
    ref.mass(q[:2], kc[:2], vc[:2], ctx[:2], None, one, RULE, table, out[:2])
    assert np.array_equal(gpu.back(d_acc, acc), np.tile(one * np.uint64(2 * calls), (b // 2, 1, 1)))
    for o in outs:
        assert np.array_equal(gpu.back(o, out), np.tile(out[:2], (b // 2, 1, 1, 1)))
