"""What the Python calls make of numbers and tensors that the C entries have no room for, without a GPU."""

import pytest

from taco_amd import hip


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
