"""The results of a scored call: which may not share memory, and which may lie side by side."""

import numpy as np
import pytest

from oracle import oracle as O
from tests.test_gpu_tree_cache import Gpu

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


def test_results_side_by_side(gpu):
    """All five in one buffer; and without alternatives, whose places do not count."""
    from tests import paged_ref as ref
    from tests.test_gpu_scores import WEIGHTS
    r = np.random.default_rng(1)
    rows, top = 5, 3
    logits, tokens = np.rint(r.standard_normal((rows, 700)) * 500).astype(np.int32), r.integers(0, 700, rows).astype(np.uint32)
    held, d = np.zeros(rows * (3 + 2 * top), np.uint32), gpu(np.zeros(rows * (3 + 2 * top), np.uint32))
    at = [d.value + 4 * rows * i for i in (0, 1, 2, 3, 3 + top)]
    gpu.hip.score_tokens(gpu.dev, gpu(logits), gpu(tokens), gpu(WEIGHTS), (rows, 700, len(WEIGHTS)), top, *at, bits=32)
    got = gpu.back(d, held).copy()
    lp, rank, entropy, tops, tops_lp = ref.scores(logits, WEIGHTS, tokens, top)
    assert np.array_equal(got[rows:2 * rows], rank)
    assert np.array_equal(got[3 * rows:(3 + top) * rows].reshape(rows, top), tops)
    ref.close(got[:rows].view(np.float32), lp, 1)
    ref.close(got[2 * rows:3 * rows].view(np.float32), entropy, 8)
    ref.close(got[(3 + top) * rows:].view(np.float32).reshape(rows, top), tops_lp, 1)
    gpu.hip.score_tokens(gpu.dev, gpu(logits), gpu(tokens), gpu(WEIGHTS), (rows, 700, len(WEIGHTS)), 0, *at[:3], at[0] + 4, at[0] + 8, bits=32)
    assert np.array_equal(gpu.back(d, held)[:3 * rows], got[:3 * rows])


def test_batch_results_that_overlap():
    from taco_amd import hip
    batch = hip.HipBatch(hip.HipModel.load(hip.HipDevice.open(0), O.build_model(O.tiny_dims(), 0x7AC0_0001, 64)), 2, 64)
    a, p, t = np.array([[0, 5], [1, 6]], np.uint32), np.full(2, hip.HS_TREE_ROOT, np.uint32), np.array([1, 2], np.uint32)
    x, y = np.zeros(2, np.float32), np.zeros((2, 2), np.uint32)
    ptr, bad = (lambda v: v.ctypes.data), hip.HS_INVALID_ARGUMENT
    assert hip.lib().hs_batch_run_scored(batch.h, ptr(a), ptr(t), 2, 2, ptr(x), None, ptr(x), ptr(y), None) == bad
    assert hip.lib().hs_batch_run_scored(batch.h, ptr(a), ptr(t), 2, 2, ptr(x), None, None, ptr(y), ptr(y) + 12) == bad
    assert batch.position(0) == 0
    assert hip.lib().hs_batch_run_scored(batch.h, ptr(a), ptr(t), 2, 0, ptr(x), None, None, ptr(x), ptr(x)) == 0
    assert batch.position(0) == 1
    assert hip.lib().hs_batch_run_tree_scored(batch.h, ptr(a), ptr(p), ptr(t), 2, 2, ptr(x), ptr(x), None, ptr(y), None) == bad
    assert hip.lib().hs_batch_run_tree_scored(batch.h, ptr(a), ptr(p), ptr(t), 2, 2, ptr(x), None, None, ptr(y), None) == 0
