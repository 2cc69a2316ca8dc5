"""Counts of the caller's that no array holds, up to the largest u32: every form of the row attention takes
the whole cache for them, as the plain 64-bit form does."""

import numpy as np
import pytest

from tests.test_gpu_tree_cache import RULE, TABLE, Gpu, check_mass, check_tree

pytestmark = pytest.mark.gpu

COUNTS = [2 ** 31, 2 ** 32 - 1, 2 ** 31 - 1, 70]
CLAMPED = (RULE[0], 8, *RULE[2:3], 53, RULE[4])  # a score shift below 13: the forms that clamp scores
LONG_TABLE = np.resize(TABLE, 20_000)            # takes the fast forms of several rows away


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


# a wave a row-head, a workgroup a row-head (head dim 64 and others), tiles, the walks over ranges, the row form
@pytest.mark.parametrize("t", [1, 20])
@pytest.mark.parametrize("hd,cap", [(64, 100), (64, 600), (32, 600), (128, 100), (128, 600), (16, 90), (80, 600),
                                    (256, 300), (64, 2100), (20, 100)])
def test_mass_counts_past_every_array(gpu, hd, cap, t):
    check_mass(gpu, 4, t, 2, hd, cap, COUNTS, [2 ** 32 - 1, t, 2 ** 31, t])
    check_mass(gpu, 4, t, 2, hd, cap, COUNTS, rule=CLAMPED)


@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("rule", [RULE, CLAMPED])
def test_mass_counts_past_every_array_in_key_chunks(gpu, hd, rule):
    """One row of few row-heads with a table that only the split decode launches take."""
    check_mass(gpu, 4, 1, 1, hd, 2100, COUNTS, rule=rule, table=LONG_TABLE)


@pytest.mark.parametrize("hd,cap", [(64, 100), (128, 600), (64, 2100), (20, 100)])
def test_tree_counts_past_every_array(gpu, hd, cap):
    check_tree(gpu, 4, 20, 2, hd, cap, COUNTS, [2 ** 32 - 1, 20, 2 ** 31, 20])
