"""The refusals of the tree, mass, evict and commit entries, without a GPU: every check comes before the
device is used, so a device that is never opened serves. And the ancestor masks of hip.tree_mask."""

import ctypes as C

import numpy as np
import pytest

from taco_amd import hip

FAKE = (C.c_char * 4096)()
BASE = (C.addressof(FAKE) + 255) // 256 * 256


class Dev:
    h = BASE


RULE = hip.AttentionRule(1, 36, 1, 59, BASE, 100, 30)


def refused(kind, fn, *args, **kw):
    with pytest.raises(hip.HipError) as e:
        fn(Dev, *args, **kw)
    assert e.value.status == kind and e.value.message
    return e.value.message


def rows(fn, q=BASE, k=BASE, v=BASE, ctx=BASE, count=BASE, third=BASE, dims=(2, 3, 2, 64, 100), rule=RULE, out=BASE, **kw):
    return lambda kind: refused(kind, fn, q, k, v, ctx, count, third, dims, rule, out, **kw)


@pytest.mark.parametrize("fn", [hip.attend_tree, hip.attend_mass])
def test_rows_refusals(fn):
    bad, unsupported = hip.HS_INVALID_ARGUMENT, hip.HS_UNSUPPORTED
    for name in ("q", "k", "v", "ctx", "third", "out"):
        rows(fn, **{name: None})(bad)
    for name in ("q", "k", "v", "ctx", "count", "third", "out"):
        rows(fn, **{name: BASE + 2})(bad)
    rows(fn, third=BASE + 4)(bad)
    rows(fn, rule=RULE._replace(attn_exp=None))(bad)
    rows(fn, rule=RULE._replace(attn_exp=BASE + 1))(bad)
    for hd in (0, 2, 66, 260):
        rows(fn, dims=(2, 3, 2, hd, 100))(unsupported)
    rows(fn, dims=(2, 3, 0, 64, 100))(unsupported)
    rows(fn, dims=(2, 3, 2, 64, 0))(unsupported)
    rows(fn, dims=(2, 3, 2, 64, (1 << 22) + 1))(unsupported)
    rows(fn, dims=(1 << 20, 1 << 10, 4, 64, 100))(unsupported)
    rows(fn, dims=(1 << 40, 3, 2, 64, 100))(unsupported)
    rows(fn, rule=RULE._replace(length=0))(unsupported)
    rows(fn, rule=RULE._replace(softmax_p=31))(unsupported)
    rows(fn, workspace=BASE + 16, workspace_bytes=1 << 40)(bad)


def test_trees_hold_256_nodes():
    rows(hip.attend_tree, dims=(2, 257, 2, 64, 1000))(hip.HS_UNSUPPORTED)


@pytest.mark.parametrize("fn", [hip.attend_tree, hip.attend_mass])
def test_nothing_to_do(fn):
    fn(Dev, BASE, BASE, BASE, BASE, None, BASE, (0, 3, 2, 64, 100), RULE, BASE)
    fn(Dev, BASE, BASE, BASE, BASE, None, BASE, (2, 0, 2, 64, 100), RULE, BASE)


def evict(k=(BASE,), v=(BASE,), mass=BASE, ctx=BASE, dims=(2, 2, 64, 100), budget=50, recent=10, mass_out=BASE,
          ctx_out=BASE + 64, kept=BASE):
    return lambda kind: refused(kind, hip.cache_evict, k, v, mass, ctx, dims, budget, recent, mass_out, ctx_out, kept)


def commit(k=(BASE,), v=(BASE,), ctx=BASE, path=BASE, accepted=BASE, dims=(2, 3, 2, 64, 100), ctx_out=BASE + 64):
    return lambda kind: refused(kind, hip.cache_commit, k, v, ctx, path, accepted, dims, ctx_out)


def test_cache_refusals():
    bad, unsupported = hip.HS_INVALID_ARGUMENT, hip.HS_UNSUPPORTED
    for f in (evict, commit):
        f(k=(None,))(bad)
        f(v=(BASE + 1,))(bad)
        f(ctx=None)(bad)
        f(ctx=BASE + 2)(bad)
        f(ctx_out=BASE + 4)(bad)  # the second count lies on the first of ctx_out
        f(ctx_out=BASE)(bad)
        f(k=(BASE, BASE))(hip.HS_LENGTH_MISMATCH)
    for hd in (0, 3, 264):
        evict(dims=(2, 2, hd, 100))(unsupported)
        commit(dims=(2, 3, 2, hd, 100))(unsupported)
    evict(dims=(1 << 30, 1 << 30, 64, 100))(unsupported)
    commit(dims=(1 << 30, 3, 1 << 30, 64, 100))(unsupported)
    evict(mass=None)(bad)
    evict(mass_out=None)(bad)
    evict(mass=BASE + 4)(bad)
    evict(mass_out=BASE + 8)(bad)  # overlaps mass in part
    for budget, recent in ((0, 0), (101, 0), (50, 51)):
        evict(budget=budget, recent=recent)(unsupported)
    commit(path=None)(bad)
    commit(accepted=None)(bad)


def test_layer_pointers():
    """A tensor of all layers and the list of its layers name the same addresses."""
    class Tensor:
        def __init__(self, shape, whole=True):
            self.shape, self.whole = shape, whole

        data_ptr = lambda self: BASE  # noqa: E731
        is_contiguous = lambda self: self.whole  # noqa: E731
        element_size = lambda self: 1  # noqa: E731
        stride = lambda self, d: int(np.prod(self.shape[d + 1:]))  # noqa: E731

    assert list(hip._dptrs(Tensor((3, 2, 2, 100, 64)))) == [BASE, BASE + 25600, BASE + 51200]
    assert len(hip._dptrs(Tensor((3, 0, 2, 100, 64)))) == 0
    with pytest.raises(ValueError):
        hip._dptrs(Tensor((3, 2, 2, 100, 64), False))


def test_tree_mask():
    m = hip.tree_mask([-1, 0, 0, 1, -1, 3])
    assert m.shape == (6, 1) and m.dtype == np.uint64
    assert [int(x) for x in m[:, 0]] == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0b101011]
    long = hip.tree_mask(list(range(-1, 69)))
    assert long.shape == (70, 2) and int(long[69, 0]) == 2 ** 64 - 1 and int(long[69, 1]) == 0b111111
    for parents in ([0], [-1, 1], [-2], [-1, 5]):
        with pytest.raises(ValueError):
            hip.tree_mask(parents)


def test_tensors_that_the_gpu_cannot_take():
    """A tensor in host memory and one with strides of its own are refused before their address is used."""
    torch = pytest.importorskip("torch")
    host = torch.zeros(4, 4, dtype=torch.int8)

    class Strided:
        is_cuda = True
        shape = (4, 4)
        data_ptr = lambda self: BASE  # noqa: E731
        is_contiguous = lambda self: False  # noqa: E731

    dims = (2, 3, 2, 64, 100)
    for x in (host, Strided()):
        for i in range(6):  # q, k, v, ctx, count, mask or accumulators
            args = [BASE] * 6
            args[i] = x
            for fn in (hip.attend_tree, hip.attend_mass):
                with pytest.raises(ValueError):
                    fn(Dev, *args, dims, RULE, BASE)
        with pytest.raises(ValueError):
            hip.attend_tree(Dev, *[BASE] * 6, dims, RULE, x)
        for k in (x, [x]):
            with pytest.raises(ValueError):
                hip.cache_commit(Dev, k, k, BASE, BASE, BASE, dims, None)
            with pytest.raises(ValueError):
                hip.cache_evict(Dev, k, k, BASE, BASE, (2, 2, 64, 100), 50, 10, BASE, None)


def test_more_rows_than_a_grid_holds():
    """2^26 rows of a head and 2^22 panels a layer are past a grid of the kernels; the workspace of a call
    that is refused, or that does nothing, is none."""
    unsupported = hip.HS_UNSUPPORTED
    for fn in (hip.attend_tree, hip.attend_mass):
        rows(fn, dims=(1 << 20, 64, 1, 64, 100))(unsupported)
        rows(fn, dims=(1 << 20, 1, 64, 64, 100))(unsupported)
    evict(dims=(1 << 20, 4, 64, 100))(unsupported)
    commit(dims=(1 << 12, 3, 1 << 10, 64, 100))(unsupported)
    sizes = hip.attend_rows_workspace
    assert sizes(8, 64, 25, 64, 8192) > 0
    for dims in ((8, 64, 25, 1 << 33, 8192), (8, 64, 25, 1 << 31, 8192), (8, 64, 25, 272, 8192), (1 << 63, 2, 1, 64, 8192),
                 (1 << 33, 1 << 33, 1, 64, 8192), (8, 64, 1 << 40, 64, 8192), (8, 64, 25, 64, 0),
                 (8, 64, 25, 64, (1 << 22) + 1), (0, 64, 25, 64, 8192), (8, 0, 25, 64, 8192), (8, 64, 0, 64, 8192),
                 (8, 64, 25, 0, 8192)):
        assert sizes(*dims) == 0, dims


def test_parents_past_32_bits():
    """They stay past the call's inputs (which is refused), and do not come round to one of them."""
    p = hip.HipBatch._parents(None, [-1, 0, 2 ** 32, 2 ** 40 + 1, 3], 5)
    assert p.dtype == np.uint32 and list(p) == [hip.HS_TREE_ROOT, 0, 5, 5, 3]
    with pytest.raises(hip.LengthMismatch):
        hip.HipBatch._parents(None, [-1], 2)
