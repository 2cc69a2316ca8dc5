"""Counts past what a call says that a stream holds: they count as that many, also with several rows."""

import numpy as np
import pytest

from tests.test_gpu_paged import check_attend
from tests.test_gpu_tree_cache import Gpu

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


@pytest.mark.parametrize("t,heads", [(1, 2), (3, 2), (7, 2), (20, 2), (70, 4)])
@pytest.mark.parametrize("keys", [64, 100, 1000, 2500, 9000])
def test_counts_past_keys(gpu, keys, t, heads):
    """The streams' pages hold more than `keys`, none of which is read: the rows count back from `keys`."""
    ctx = np.array([keys + 1, keys + 500, 2 ** 32 - 1, keys, 2 ** 31], np.uint32)
    check_attend(gpu, 5, t, heads, 2, 64, 128, keys, ctx, [t, max(1, t // 2), t, t, 0], holes=0.05, seed=keys + t)
    check_attend(gpu, 5, t, heads, 2, 64, 16, keys, ctx, None, seed=keys + t)
