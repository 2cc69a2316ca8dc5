"""Every form of the eviction against the plain form: each capacity class by copies of 16 bytes and of 4, with head dims
whose rows do not divide the workgroup, and caches 4 bytes off a multiple of 16 (evictions and commits)."""

import ctypes as C

import numpy as np
import pytest

from tests import attention_ref as ref
from tests.test_gpu_tree_cache import Gpu, caches, check_evict

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


@pytest.mark.parametrize("hd", [4, 20, 80, 192, 252, 256])
@pytest.mark.parametrize("cap,budget,recent", [(1000, 700, 90), (3000, 1000, 333), (4097, 4000, 0), (9000, 2000, 2000),
                                               (17_000, 6000, 511), (20_000, 19_000, 4001)])
def test_capacities_and_words(gpu, hd, cap, budget, recent):
    check_evict(gpu, 1, 2, 1, hd, cap, [cap, budget + 1], budget, recent, alias=hd % 8 == 0)


@pytest.mark.parametrize("hd,cap", [(64, 700), (256, 3000), (128, 9000), (64, 17_000)])
def test_unaligned_caches(gpu, hd, cap):
    print(f"unaligned caches, head dim {hd}, cap {cap}", flush=True)
    r, (b, h, t) = np.random.default_rng(hd + cap), (2, 1, 40)
    budget, recent = cap // 2, cap // 7
    kc, vc = caches(r, b, h, cap, hd)

    def inside(x):
        big = np.full(x.nbytes + 64, 55, np.int8)
        big[4:4 + x.nbytes] = x.ravel()
        p = gpu(big)
        return big, p, C.c_void_p(p.value + 4)

    held = [inside(kc), inside(vc)]
    ptrs = [[x[2]] for x in held]
    ctx, accepted = np.array([cap - t, 3], np.uint32), np.array([7, 9], np.uint32)
    path = np.zeros((b, t), np.uint32)
    for s in range(b):
        path[s, :accepted[s]] = np.sort(r.permutation(t)[:accepted[s]])
    after, cut = np.zeros(b, np.uint32), np.zeros(b, np.uint32)
    d_after, d_cut = gpu(after), gpu(cut)
    gpu.hip.cache_commit(gpu.dev, *ptrs, gpu(ctx), gpu(path), gpu(accepted), (b, t, h, hd, cap), d_after)
    ref.commit([kc], [vc], ctx, path, accepted, after)
    acc = r.integers(0, 50, (1, b, h, cap)).astype(np.uint64)
    d_acc = gpu(acc)
    gpu.hip.cache_evict(gpu.dev, *ptrs, d_acc, d_after, (b, h, hd, cap), budget, recent, d_acc, d_cut)
    ref.evict([kc], [vc], acc, after, budget, recent, acc, cut, None)
    for d, x in ((d_after, after), (d_cut, cut), (d_acc, acc)):
        assert np.array_equal(gpu.back(d, x), x)
    for (big, p, _), x in zip(held, (kc, vc)):
        got = gpu.back(p, big)
        assert np.array_equal(got[4:4 + x.nbytes].reshape(x.shape), x)
        assert (got[:4] == 55).all() and (got[4 + x.nbytes:] == 55).all()
