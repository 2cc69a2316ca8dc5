"""What the Python calls make of numbers and tensors that the C entries have no room for, without a GPU."""

import ctypes as C

import numpy as np
import pytest

from taco_amd import hip

LAST = 2 ** 32 - 1


@pytest.mark.parametrize("x,want", [([], []), ([0, 7, LAST], [0, 7, LAST]), ([2 ** 32], [LAST]), ([-1, 2 ** 80, 5], [LAST, LAST, 5]),
                                    ([np.int64(2 ** 32 + 3), 1], [LAST, 1]), (np.array([-2, 2 ** 40, 6]), [LAST, LAST, 6]),
                                    (np.array([2 ** 63, 6], np.uint64), [LAST, 6]), (np.array([3, 4], np.uint8), [3, 4])])
def test_numbers_past_32_bits(x, want):
    """They become 2^32 - 1, which the library refuses, and do not come round to a slot, token or node."""
    got = hip._u32(x)
    assert got.dtype == np.uint32 and got.tolist() == want and got.flags.c_contiguous


def test_inputs_and_queries_past_32_bits():
    assert hip._inputs([(np.int64(2 ** 32), 5), (1, np.int64(2 ** 32 + 9))]).tolist() == [[LAST, 5], [1, LAST]]
    assert hip._inputs([]).shape == hip._queries([]).shape == (0, 2)
    assert hip._queries([(0, 5), (1, LAST)]).tolist() == [[0, 5], [1, LAST]]
    for bad in ([(0, 2 ** 32 + 5)], [(0, np.int64(2 ** 32 + 5))], np.array([[1, -1]]), [(2 ** 70, 1)]):
        with pytest.raises(hip.Unsupported):
            hip._queries(bad)


def test_paths_past_32_bits(monkeypatch):
    calls = []

    class Library:
        def hs_batch_commit_paths(self, h, slots, lengths, paths, n):
            def array(p, count):
                return np.ctypeslib.as_array(C.cast(p, C.POINTER(C.c_uint32)), (count,)).tolist() if count else []
            counts = array(lengths, n)
            calls.append((array(slots, n), counts, array(paths, sum(counts))))
            return hip.HS_OK

    monkeypatch.setattr(hip, "lib", lambda: Library())
    batch = hip.HipBatch.__new__(hip.HipBatch)
    batch.h = None
    batch.commit_paths({np.int64(2 ** 32): [0], 3: [np.int64(2 ** 32), 1], 2: []})
    batch.commit_paths({})
    assert calls == [([LAST, 3, 2], [1, 2, 0], [0, LAST, 1]), ([], [], [])]


def test_one_layer_whose_stride_says_nothing():
    """The stride of an axis of one is free: with a stride of 0 the layer was not passed at all."""
    torch = pytest.importorskip("torch")
    whole = torch.zeros(2, 3, 5, 4, dtype=torch.int8)

    class OnGpu:
        is_cuda = True

        def __init__(self, x):
            self.x = x

        def __getattr__(self, name):
            return getattr(self.x, name)

    for stride in (0, 1, 120):
        one = whole.as_strided((1, 2, 3, 5, 4), (stride, 60, 20, 4, 1))
        assert one.is_contiguous()
        assert list(hip._dptrs(OnGpu(one))) == [whole.data_ptr()]
    assert list(hip._dptrs(OnGpu(whole))) == [whole.data_ptr(), whole.data_ptr() + 60]
    assert len(hip._dptrs(OnGpu(whole[:0]))) == 0


def test_rules_that_a_call_would_cut():
    rule = hip.AttentionRule(-2 ** 31, 255, 2 ** 31 - 1, 0, 4096, 100, 30)
    assert rule == (-2 ** 31, 255, 2 ** 31 - 1, 0, 4096, 100, 30) and rule._replace(softmax_p=31).softmax_p == 31
    for change in ({"score_m": 2 ** 31}, {"out_m": -2 ** 31 - 1}, {"score_s": 256}, {"score_s": -1}, {"out_s": 292},
                   {"softmax_p": 286}, {"length": -1}, {"length": 2 ** 64}):
        with pytest.raises(hip.Unsupported):
            rule._replace(**change)
        with pytest.raises(hip.Unsupported):
            hip.AttentionRule(**{**rule._asdict(), **change})


@pytest.mark.parametrize("parents,want", [([-1, 0, 1], [LAST, 0, 1]), ([hip.HS_TREE_ROOT, -1, 2], [LAST, LAST, 2]),
                                          ([-2, -2 ** 63, -1], [3, 3, LAST]), ([2 ** 63, 2 ** 80, -2 ** 80], [3, 3, 3]),
                                          (np.array([2 ** 64 - 1, 2 ** 63, 1], np.uint64), [3, 3, 1]),
                                          (np.array([LAST, 1, 3], np.uint32), [LAST, 1, 3])])
def test_parents_that_are_none(parents, want):
    """Only -1 and HS_TREE_ROOT are the root; what is neither that nor an input stays none."""
    got = hip.HipBatch._parents(None, parents, 3)
    assert got.dtype == np.uint32 and got.tolist() == want
