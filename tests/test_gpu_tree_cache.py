"""Attention of trees of drafted tokens, attention with accumulated weights, eviction and path commits
against the plain 64-bit forms of attention_ref.py, value for value: head dims with and without a fast form,
row counts around the tiles, contexts from none to the whole cache, ragged counts, masks that leave
rows empty, every shape of rule, and a serving loop of all four."""

import ctypes as C

import numpy as np
import pytest

from tests import attention_ref as ref

pytestmark = pytest.mark.gpu

TABLE = np.array([round(2 ** 30 * np.exp(-i / 256)) for i in range(8192)], np.int32)
RULE = (1_400_000_000, 36, 1_300_000_000, 59, 30)


class Gpu:
    """Device copies of host arrays; `back` reads one again."""

    def __init__(self):
        from taco_amd import hip
        self.hip, self.dev, self.held = hip, hip.HipDevice.open(0), []

    def __call__(self, x):
        x = np.ascontiguousarray(x)
        p = C.c_void_p()
        self.hip._check(self.hip.lib().hs_device_alloc(self.dev.h, max(x.nbytes, 16), C.byref(p)))
        self.held.append(p)
        if x.nbytes:
            self.hip._check(self.hip.lib().hs_device_upload(self.dev.h, p, self.hip._ptr(x), x.nbytes))
        return p

    def back(self, p, like):
        out = np.empty_like(like)
        self.hip._check(self.hip.lib().hs_device_download(self.dev.h, self.hip._ptr(out), p, out.nbytes))
        return out

    def rule(self, rule, table):
        return self.hip.AttentionRule(*rule[:4], self(table), len(table), rule[4])

    def free(self):
        for p in self.held:
            self.hip.lib().hs_device_free(self.dev.h, p)
        self.held = []


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


def caches(r, b, h, cap, hd, most=128):
    return [r.integers(-most, most, (b, h, cap, hd)).astype(np.int8) for _ in range(2)]


def masks(gpu, r, b, t, empty=0.0):
    m = np.stack([gpu.hip.tree_mask(ref.random_parents(r, t)) for _ in range(b)])
    m[r.random((b, t)) < empty] = 0
    return m


def check_tree(gpu, b, t, h, hd, cap, ctx, nodes=None, rule=RULE, table=TABLE, seed=1, empty=0.0, full=False):
    print(f"tree {b}x{t}x{h}x{hd} cap {cap}", flush=True)
    r = np.random.default_rng(seed)
    q = r.integers(-128, 128, (b, t, h, hd)).astype(np.int8)
    kc, vc = caches(r, b, h, cap, hd)
    ctx = np.resize(np.array(ctx, np.uint32), b)
    nodes = None if nodes is None else np.resize(np.array(nodes, np.uint32), b)
    mask = masks(gpu, r, b, t, empty)
    if full:  # every bit set, those behind the tree too
        mask[:] = np.uint64(2 ** 64 - 1)
    out = np.full((b, t, h, hd), 77, np.int8)
    d_out = gpu(out)
    gpu.hip.attend_tree(gpu.dev, gpu(q), gpu(kc), gpu(vc), gpu(ctx), None if nodes is None else gpu(nodes), gpu(mask),
                        (b, t, h, hd, cap), gpu.rule(rule, table), d_out)
    got = gpu.back(d_out, out)
    assert np.array_equal(got, ref.tree(q, kc, vc, ctx, nodes, mask, rule, table, out))


def check_mass(gpu, b, t, h, hd, cap, ctx, rows=None, rule=RULE, table=TABLE, seed=2, start=0):
    print(f"mass {b}x{t}x{h}x{hd} cap {cap}", flush=True)
    r = np.random.default_rng(seed)
    q = r.integers(-128, 128, (b, t, h, hd)).astype(np.int8)
    kc, vc = caches(r, b, h, cap, hd)
    ctx = np.resize(np.array(ctx, np.uint32), b)
    rows = None if rows is None else np.resize(np.array(rows, np.uint32), b)
    acc = np.full((b, h, cap), start, np.uint64)
    out = np.full((b, t, h, hd), 77, np.int8)
    d_out, d_acc = gpu(out), gpu(acc)
    args = (gpu.dev, gpu(q), gpu(kc), gpu(vc), gpu(ctx), None if rows is None else gpu(rows), d_acc,
            (b, t, h, hd, cap), gpu.rule(rule, table), d_out)
    for _ in range(2):  # the second call adds the same again
        gpu.hip.attend_mass(*args)
        ref.mass(q, kc, vc, ctx, rows, acc, rule, table, out)
        assert np.array_equal(gpu.back(d_out, out), out)
        assert np.array_equal(gpu.back(d_acc, acc), acc)


HEAD_DIMS = [4, 16, 20, 32, 48, 64, 80, 128, 192, 256]


@pytest.mark.parametrize("hd", HEAD_DIMS)
def test_tree_head_dims(gpu, hd):
    check_tree(gpu, 5, 19, 3, hd, 300, [0, 281, 63, 64, 200], [19, 17, 1, 0, 5])


@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 33, 63, 64, 65, 128, 200, 256])
def test_tree_sizes(gpu, t):
    check_tree(gpu, 4, t, 2, 64, 400, [0, 400 - t, 65, 1], [t, t, (t + 1) // 2, t], empty=0.1)


@pytest.mark.parametrize("cap,ctx", [(1, [0]), (64, [63, 0]), (65, [64, 1]), (257, [240, 255, 0]), (1024, [1000, 1, 0]),
                                     (1025, [1009]), (2049, [2030, 700]), (4096, [4080, 1500]), (4100, [4050, 100]),
                                     (9000, [8970, 4096, 0])])
def test_tree_contexts(gpu, cap, ctx):
    t = min(16, cap - max(ctx))
    check_tree(gpu, len(ctx) + 1, t, 2, 64, cap, ctx)


@pytest.mark.parametrize("hd,cap", [(32, 5000), (80, 2300), (128, 4500), (256, 3000), (20, 700)])
def test_tree_long_contexts_of_other_head_dims(gpu, hd, cap):
    check_tree(gpu, 2, 18, 2, hd, cap, [cap - 18, cap // 2])


@pytest.mark.parametrize("t", [1, 16, 17, 33, 64, 90, 256])
def test_tree_sizes_over_long_contexts(gpu, t):
    check_tree(gpu, 3, t, 2, 64, 2600, [2600 - t, 300, 0], [t, (t + 1) // 2, t], empty=0.1)


@pytest.mark.parametrize("hd", [16, 80, 256])
def test_many_long_contexts(gpu, hd):
    """So many streams that a workgroup walks a whole cache by itself."""
    check_tree(gpu, 400 if hd == 16 else 128, 3, 4 if hd == 16 else 13, hd, 2052, [2049, 5, 2000, 0])
    check_mass(gpu, 128, 3, 13, hd, 2052, [2049, 5, 2000, 3], seed=hd)


@pytest.mark.parametrize("hd", [20, 64, 128])
def test_tree_rows_that_see_nothing(gpu, hd):
    """No context and empty masks: rows of zeros; every bit set: only the stream's own nodes count."""
    check_tree(gpu, 3, 20, 2, hd, 100, [0], [20, 7, 0], empty=1.0)
    check_tree(gpu, 3, 20, 2, hd, 100, [0, 50], [20, 7, 1], full=True)


def test_tree_counts_beyond_the_cache(gpu):
    """Counts larger than the arrays: t rows at most, and no key past the cache."""
    check_tree(gpu, 4, 20, 2, 64, 100, [95, 100, 4000, 10], [20, 20, 20, 1000])


RULES = [(1_400_000_000, 8, 1_300_000_000, 53, 30),   # scores beyond +-2^40
         (-1_400_000_000, 34, -1_300_000_000, 60, 30), (2 ** 31 - 1, 0, 2 ** 31 - 1, 0, 30),
         (1 << 30, 22, 1 << 30, 48, 30), (1 << 30, 21, 1 << 30, 47, 16), (1 << 30, 40, 1 << 30, 30, 1),
         (1 << 30, 62, 1 << 30, 63, 30), (1 << 30, 90, 1 << 30, 95, 30), (1 << 30, 36, 1 << 30, 96, 30),
         (1 << 30, 36, 1 << 30, 28, 0), (-2 ** 31, 36, -2 ** 31, 64, 30)]


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("hd", [64, 128])
def test_rules(gpu, rule, hd):
    check_tree(gpu, 2, 18, 2, hd, 330, [300, 20], rule=rule)
    check_mass(gpu, 2, 18, 2, hd, 330, [330, 20], rule=rule)
    check_mass(gpu, 2, 1, 2, hd, 330, [330, 20], rule=rule)


@pytest.mark.parametrize("table", [TABLE[:1], TABLE[:700], np.resize(TABLE, 20_000), np.zeros(5, np.int32),
                                   np.array([0, 0, 7, 2 ** 31 - 1], np.int32)])
def test_tables(gpu, table):
    """One entry, a cut tail, one longer than the copy on the chip, and tables whose entries at the top are 0."""
    check_tree(gpu, 2, 18, 2, 64, 330, [300, 20], table=table)
    check_mass(gpu, 2, 5, 2, 64, 330, [330, 20], table=table)
    check_mass(gpu, 2, 1, 2, 64, 330, [330, 20], table=table)
    check_tree(gpu, 1, 18, 1, 64, 4500, [4400], table=table)


@pytest.mark.parametrize("hd", HEAD_DIMS)
@pytest.mark.parametrize("t", [1, 3, 40])
def test_mass_head_dims(gpu, hd, t):
    check_mass(gpu, 5, t, 3, hd, 300, [300, 64, 65, 255, 44], None if t == 1 else [t, 1, 0, t - 1, t])


@pytest.mark.parametrize("cap", [1, 63, 64, 65, 128, 257, 512, 600, 1024, 1025, 2048, 2500, 4097, 9000])
@pytest.mark.parametrize("hd", [64, 128])
def test_mass_steps(gpu, cap, hd):
    check_mass(gpu, 3, 1, 2, hd, cap, [cap, (cap + 1) // 2, 1])


@pytest.mark.parametrize("t,cap", [(2, 2), (16, 1024), (17, 1100), (64, 64), (100, 100), (130, 700), (33, 4200), (40, 9000),
                                   (1100, 2600), (1100, 1900)])
def test_mass_chunks(gpu, t, cap):
    check_mass(gpu, 3, t, 2, 64, cap, [cap, t, (cap + t) // 2], [t, t, max(1, t // 2)])


def test_long_table_over_a_long_cache(gpu):
    """A table longer than the fast forms take, and the workspace that attend_rows_workspace names for it."""
    table = np.resize(TABLE, 20_000)
    for t in (1, 3):
        check_mass(gpu, 2, t, 2, 64, 2500, [2500, 700], table=table)
    r = np.random.default_rng(3)
    q, (kc, vc) = r.integers(-128, 128, (2, 1, 2, 64)).astype(np.int8), caches(r, 2, 2, 2500, 64)
    ctx, acc, out = np.array([2400, 9], np.uint32), np.zeros((2, 2, 2500), np.uint64), np.zeros_like(q)
    d_out, need = gpu(out), gpu.hip.attend_rows_workspace(2, 1, 2, 64, 2500)
    gpu.hip.attend_mass(gpu.dev, gpu(q), gpu(kc), gpu(vc), gpu(ctx), None, gpu(acc), (2, 1, 2, 64, 2500),
                        gpu.rule(RULE, table), d_out, gpu(np.zeros(need, np.uint8)), need)
    ref.mass(q, kc, vc, ctx, None, acc, RULE, table, out)
    assert np.array_equal(gpu.back(d_out, out), out)


def test_unaligned_rows_and_caches(gpu):
    """Arrays 4 bytes off a multiple of 16 (the caller's slices): the row form, the same values; and queries,
    caches and outputs inside larger arrays, whose other bytes stay."""
    r = np.random.default_rng(8)
    b, t, h, hd, cap = 2, 6, 2, 64, 90
    q, (kc, vc) = r.integers(-128, 128, (b, t, h, hd)).astype(np.int8), caches(r, b, h, cap, hd)
    ctx, mask = np.array([70, 3], np.uint32), masks(gpu, r, b, t)
    out, acc = np.zeros_like(q), np.zeros((b, h, cap), np.uint64)

    def inside(x):
        big = np.full(x.nbytes + 64, 55, np.int8)
        big[4:4 + x.nbytes] = np.frombuffer(x.tobytes(), np.int8)
        p = gpu(big)
        return big, p, C.c_void_p(p.value + 4)

    held = [inside(x) for x in (q, kc, vc, out)]
    rule = gpu.rule(RULE, TABLE)
    ptrs = [x[2] for x in held]
    gpu.hip.attend_tree(gpu.dev, *ptrs[:3], gpu(ctx), None, gpu(mask), (b, t, h, hd, cap), rule, ptrs[3])
    ref.tree(q, kc, vc, ctx, None, mask, RULE, TABLE, out)
    big = gpu.back(held[3][1], held[3][0])
    assert np.array_equal(big[4:4 + out.nbytes].reshape(out.shape), out)
    assert (big[:4] == 55).all() and (big[4 + out.nbytes:] == 55).all()
    d_acc = gpu(acc)
    keys = ctx + np.uint32(t)
    gpu.hip.attend_mass(gpu.dev, *ptrs[:3], gpu(keys), None, d_acc, (b, t, h, hd, cap), rule, ptrs[3])
    ref.mass(q, kc, vc, keys, None, acc, RULE, TABLE, out)
    assert np.array_equal(gpu.back(d_acc, acc), acc)
    one = gpu(np.ones(b, np.uint32))
    gpu.hip.attend_mass(gpu.dev, *ptrs[:3], gpu(keys), one, d_acc, (b, 1, h, hd, cap), rule, ptrs[3])
    first = np.zeros((b, 1, h, hd), np.int8)
    ref.mass(q.reshape(b * t, h, hd)[:b, None], kc, vc, keys, None, acc, RULE, TABLE, first)
    assert np.array_equal(gpu.back(d_acc, acc), acc)


def test_many_panels(gpu):
    """More workgroups than fit at once, some streams without a row."""
    check_tree(gpu, 300, 20, 4, 16, 90, [70, 0, 33], [20, 0, 17, 3])
    check_mass(gpu, 300, 2, 4, 16, 90, [70, 2, 33, 0], [2, 0, 1, 2])
    check_mass(gpu, 700, 1, 4, 16, 600, [70, 0, 333, 600], [1, 1, 0, 1])
    check_tree(gpu, 130, 40, 5, 16, 1100, [1060, 0, 33], [40, 0, 17, 3])
    check_mass(gpu, 130, 1, 4, 16, 2100, [2100, 0, 333, 2049, 1], [1, 1, 0, 1])


def test_mass_counts_beyond_the_cache(gpu):
    """More rows than keys: the first ones see nothing. Counts past the arrays. No row at all."""
    check_mass(gpu, 4, 20, 2, 64, 100, [5, 0, 4000, 100], [20, 20, 20, 0], start=2 ** 40)


def check_evict(gpu, layers, b, h, hd, cap, ctx, budget, recent, acc=None, seed=3, alias=False, with_kept=True):
    print(f"evict {layers}x{b}x{h}x{hd} cap {cap} budget {budget} recent {recent}", flush=True)
    r = np.random.default_rng(seed)
    ks, vs = zip(*[caches(r, b, h, cap, hd) for _ in range(layers)])
    ks, vs = list(ks), list(vs)
    ctx = np.resize(np.array(ctx, np.uint32), b)
    if acc is None:
        acc = (np.exp(2 * r.standard_normal((layers, b, h, cap))) * 2 ** 28).astype(np.uint64)
        acc[r.random(acc.shape) < 0.1] = 0
    acc = np.ascontiguousarray(np.broadcast_to(acc, (layers, b, h, cap))).astype(np.uint64)
    acc_out = acc if alias else np.full(acc.shape, 9, np.uint64)
    ctx_out, kept = np.full(b, 99, np.uint32), np.full((layers, b, h, budget), 4_000_000_000, np.uint32)
    dk, dv, d_acc = [gpu(x) for x in ks], [gpu(x) for x in vs], gpu(acc)
    d_acc_out = d_acc if alias else gpu(acc_out)
    d_ctx_out, d_kept = gpu(ctx_out), gpu(kept)
    gpu.hip.cache_evict(gpu.dev, dk, dv, d_acc, gpu(ctx), (b, h, hd, cap), budget, recent, d_acc_out, d_ctx_out,
                        d_kept if with_kept else None)
    ref.evict(ks, vs, acc, ctx, budget, recent, acc_out, ctx_out, kept if with_kept else None)
    for d, x in zip(dk + dv + [d_acc, d_acc_out, d_ctx_out, d_kept], ks + vs + [acc, acc_out, ctx_out, kept]):
        assert np.array_equal(gpu.back(d, x), x)


@pytest.mark.parametrize("hd", HEAD_DIMS)
def test_evict_head_dims(gpu, hd):
    check_evict(gpu, 2, 4, 2, hd, 200, [200, 199, 90, 91], 90, 30)


@pytest.mark.parametrize("cap,budget,recent", [(1, 1, 0), (2, 1, 0), (2, 1, 1), (300, 299, 0), (300, 1, 0), (300, 64, 64),
                                               (1024, 512, 128), (1024, 1023, 700), (700, 300, 299), (3000, 1000, 100), (5000, 1300, 17), (16384, 9000, 1000),
                                               (20000, 6000, 511), (20000, 300, 0)])
@pytest.mark.parametrize("alias", [False, True])
def test_evict_budgets(gpu, cap, budget, recent, alias):
    check_evict(gpu, 1, 3, 2, 64, cap, [cap, budget, min(cap, budget + 1)], budget, recent, alias=alias)


@pytest.mark.parametrize("acc", [0, 5, 2 ** 64 - 1])
def test_evict_ties_go_to_the_lowest_index(gpu, acc):
    check_evict(gpu, 1, 2, 2, 64, 900, [900, 700], 400, 50, acc=np.uint64(acc))


def test_evict_orders_of_weights(gpu):
    """Rising and falling weights (every kept key moves, none does), two values only, the top bits alone."""
    i = np.arange(1500, dtype=np.uint64)
    for acc in (i, 1500 - i, i % 2, i % 7, i * i * i, i << np.uint64(20), (i % 3) << np.uint64(62), np.where(i == 700, 2 ** 63, i).astype(np.uint64)):
        check_evict(gpu, 1, 2, 1, 64, 1500, [1500, 1100], 600, 100, acc=acc)


def test_evict_many_layers_and_no_list(gpu):
    check_evict(gpu, 70, 2, 1, 16, 40, [40, 21], 20, 5, with_kept=False)


def check_commit(gpu, layers, b, h, hd, cap, t, ctx, accepted, path=None, seed=4):
    print(f"commit {layers}x{b}x{t}x{h}x{hd} cap {cap}", flush=True)
    r = np.random.default_rng(seed)
    ks, vs = zip(*[caches(r, b, h, cap, hd) for _ in range(layers)])
    ks, vs = list(ks), list(vs)
    ctx, accepted = np.resize(np.array(ctx, np.uint32), b), np.resize(np.array(accepted, np.uint32), b)
    if path is None:
        path = np.full((b, t), 4_000_000_000, np.uint32)  # entries past the accepted ones are never read
        for s in range(b):
            path[s, :accepted[s]] = np.sort(r.permutation(t)[:accepted[s]])
    path = np.array(path, np.uint32)
    ctx_out = np.full(b, 99, np.uint32)
    dk, dv, d_ctx_out = [gpu(x) for x in ks], [gpu(x) for x in vs], gpu(ctx_out)
    gpu.hip.cache_commit(gpu.dev, dk, dv, gpu(ctx), gpu(path), gpu(accepted), (b, t, h, hd, cap), d_ctx_out)
    ref.commit(ks, vs, ctx, path, accepted, ctx_out)
    for d, x in zip(dk + dv + [d_ctx_out], ks + vs + [ctx_out]):
        assert np.array_equal(gpu.back(d, x), x)


@pytest.mark.parametrize("hd", HEAD_DIMS)
def test_commit_head_dims(gpu, hd):
    check_commit(gpu, 2, 5, 3, hd, 120, 30, [0, 90, 7, 50, 1], [30, 0, 1, 12, 29])


@pytest.mark.parametrize("t", [1, 2, 64, 256, 1000])
def test_commit_sizes(gpu, t):
    check_commit(gpu, 3, 4, 2, 64, t + 50, t, [0, 50, 13, 50], [t, t, (t + 1) // 2, 1])


def test_commit_same_node_twice_and_many_layers(gpu):
    check_commit(gpu, 66, 2, 1, 64, 40, 6, [3, 30], [3, 4], path=[[2, 2, 5, 0, 0, 0], [0, 4, 4, 4, 0, 0]])


def test_serving_loop(gpu):
    """A prompt in causal chunks, then rounds of: a tree of drafts, the accepted path, a decode step, and
    the caches cut to their budget when they outgrow it."""
    r = np.random.default_rng(11)
    b, h, hd, cap, t, budget, recent = 4, 3, 64, 160, 12, 96, 24
    kc, vc = caches(r, b, h, cap, hd)
    acc, table = np.zeros((1, b, h, cap), np.uint64), TABLE
    dk, dv, d_acc, rule = gpu(kc), gpu(vc), gpu(acc), gpu.rule(RULE, table)
    ctx, spare = gpu(np.zeros(b, np.uint32)), gpu(np.zeros(b, np.uint32))
    n = np.zeros(b, np.uint32)

    def append(count):
        """The new tokens' rows at their places, here and on the GPU."""
        new_k, new_v = caches(r, b, h, int(max(count)), hd)
        k, v = gpu.back(dk, kc), gpu.back(dv, vc)
        assert np.array_equal(k, kc) and np.array_equal(v, vc)
        for s in range(b):
            kc[s, :, n[s]:n[s] + count[s]] = new_k[s, :, :count[s]]
            vc[s, :, n[s]:n[s] + count[s]] = new_v[s, :, :count[s]]
        for d, x in ((dk, kc), (dv, vc)):
            gpu.hip._check(gpu.hip.lib().hs_device_upload(gpu.dev.h, d, gpu.hip._ptr(x), x.nbytes))

    def causal(rows):
        q = r.integers(-128, 128, (b, int(max(rows)), h, hd)).astype(np.int8)
        out = np.zeros_like(q)
        d_out = gpu(out)
        gpu.hip.attend_mass(gpu.dev, gpu(q), dk, dv, gpu(n), gpu(rows), d_acc, (*q.shape, cap), rule, d_out)
        ref.mass(q, kc, vc, n, rows, acc[0], RULE, table, out)
        assert np.array_equal(gpu.back(d_out, out), out)
        assert np.array_equal(gpu.back(d_acc, acc), acc)

    for chunk in ([40, 33, 20, 50], [37, 40, 1, 0]):
        rows = np.array(chunk, np.uint32)
        append(rows)
        n += rows
        causal(rows)
    for _ in range(9):
        gpu.hip._check(gpu.hip.lib().hs_device_upload(gpu.dev.h, ctx, gpu.hip._ptr(n), n.nbytes))
        nodes = r.integers(1, t + 1, b).astype(np.uint32)
        append(nodes)
        q, mask = r.integers(-128, 128, (b, t, h, hd)).astype(np.int8), np.zeros((b, t, 1), np.uint64)
        parents = [ref.random_parents(r, t) for _ in range(b)]
        path, accepted = np.zeros((b, t), np.uint32), np.zeros(b, np.uint32)
        for s in range(b):
            mask[s] = gpu.hip.tree_mask(parents[s])
            at, chain = int(r.integers(0, nodes[s])), []
            while at >= 0:
                chain.insert(0, at)
                at = parents[s][at]
            path[s, :len(chain)], accepted[s] = chain, len(chain)
        out = np.zeros_like(q)
        d_out = gpu(out)
        gpu.hip.attend_tree(gpu.dev, gpu(q), dk, dv, ctx, gpu(nodes), gpu(mask), (b, t, h, hd, cap), rule, d_out)
        ref.tree(q, kc, vc, n, nodes, mask, RULE, table, out)
        assert np.array_equal(gpu.back(d_out, out), out)
        gpu.hip.cache_commit(gpu.dev, [dk], [dv], ctx, gpu(path), gpu(accepted), (b, t, h, hd, cap), spare)
        m = np.zeros_like(n)
        ref.commit([kc], [vc], n, path, accepted, m)
        n = m
        assert np.array_equal(gpu.back(spare, n), n)
        one = np.ones(b, np.uint32)
        append(one)
        n = n + one
        causal(one)
        gpu.hip._check(gpu.hip.lib().hs_device_upload(gpu.dev.h, spare, gpu.hip._ptr(n), n.nbytes))
        gpu.hip.cache_evict(gpu.dev, [dk], [dv], d_acc, spare, (b, h, hd, cap), budget, recent, d_acc, ctx)
        m = np.zeros_like(n)
        ref.evict([kc], [vc], acc, n, budget, recent, acc, m, None)
        n = m
        assert np.array_equal(gpu.back(ctx, n), n) and np.array_equal(gpu.back(d_acc, acc), acc)
    assert n.max() == budget


def test_plane_sums_of_many_keys(gpu):
    """133,151 keys and more of equal weight, p = 8,064, whose lowest digit is -128, over values of -128: a digit plane's
    sum over all of them passes 2^31, so no wave may add up that many (520 panels: enough for one launch else)."""
    b, t, hd, ctx = 520, 40, 16, 133_150
    cap = ctx + t
    count, keys = np.zeros(b, np.uint32), np.zeros(b, np.uint32)
    count[-1], keys[-1] = t, ctx
    r = np.random.default_rng(2)
    mask = np.zeros((b, t, 1), np.uint64)
    mask[-1] = masks(gpu, r, 1, t)[0]
    q = np.zeros((b, t, 1, hd), np.int8)
    v = np.full((1, 1, cap, hd), -128, np.int8)
    panels = []
    for x in (np.zeros_like(v), v):
        p = C.c_void_p()
        gpu.hip._check(gpu.hip.lib().hs_device_alloc(gpu.dev.h, b * x.nbytes, C.byref(p)))
        gpu.held.append(p)
        gpu.hip._check(gpu.hip.lib().hs_device_upload(gpu.dev.h, C.c_void_p(p.value + (b - 1) * x.nbytes), gpu.hip._ptr(x), x.nbytes))
        panels.append(p)
    rule = (1 << 30, 36, 1 << 30, 60, 30)
    out = np.full(q.shape, 77, np.int8)
    d_out = gpu(out)
    gpu.hip.attend_tree(gpu.dev, gpu(q), *panels, gpu(keys), gpu(count), gpu(mask), (b, t, 1, hd, cap), gpu.rule(rule, TABLE), d_out)
    ref.tree(q[-1:], np.zeros_like(v), v, keys[-1:], None, mask[-1:], rule, TABLE, out[-1:])
    assert np.array_equal(gpu.back(d_out, out), out) and (out[-1] < -100).all()


def test_caches_of_more_than_4_gib(gpu):
    """The last of 257 streams of 2 heads and 131,072 places: its panels lie past 2^32 bytes."""
    r = np.random.default_rng(21)
    b, t, h, hd, cap, budget, recent = 257, 5, 2, 64, 131_072, 1000, 100
    L = gpu.hip.lib()
    kc, vc = caches(r, 1, h, cap, hd)
    whole = []
    for x in (kc, vc):
        p = C.c_void_p()
        gpu.hip._check(L.hs_device_alloc(gpu.dev.h, b * x.nbytes, C.byref(p)))
        gpu.held.append(p)
        last = C.c_void_p(p.value + (b - 1) * x.nbytes)
        gpu.hip._check(L.hs_device_upload(gpu.dev.h, last, gpu.hip._ptr(x), x.nbytes))
        whole.append((p, last))
    (dk, last_k), (dv, last_v) = whole
    q = r.integers(-128, 128, (b, t, h, hd)).astype(np.int8)
    ctx, count = np.zeros(b, np.uint32), np.zeros(b, np.uint32)
    ctx[-1], count[-1] = cap - t, t
    mask = np.zeros((b, t, 1), np.uint64)
    mask[-1] = masks(gpu, r, 1, t)[0]
    out, acc = np.zeros_like(q), np.zeros((1, b, h, cap), np.uint64)
    d_out, d_acc, rule = gpu(out), gpu(acc), gpu.rule(RULE, TABLE)
    gpu.hip.attend_tree(gpu.dev, gpu(q), dk, dv, gpu(ctx), gpu(count), gpu(mask), (b, t, h, hd, cap), rule, d_out)
    ref.tree(q[-1:], kc, vc, ctx[-1:], None, mask[-1:], RULE, TABLE, out[-1:])
    assert np.array_equal(gpu.back(d_out, out), out)
    keys = ctx + count
    for rows, n in ((t, count), (1, np.minimum(count, 1))):  # a chunk of rows, then one row a stream
        first = np.ascontiguousarray(q[:, :rows])
        out = np.zeros_like(first)
        d_out = gpu(out)
        gpu.hip.attend_mass(gpu.dev, gpu(first), dk, dv, gpu(keys), gpu(n), d_acc, (b, rows, h, hd, cap), rule, d_out)
        ref.mass(first[-1:], kc, vc, keys[-1:], None, acc[0, -1:], RULE, TABLE, out[-1:])
        assert np.array_equal(gpu.back(d_out, out), out)
        assert np.array_equal(gpu.back(d_acc, acc), acc)
    path, accepted = np.zeros((b, t), np.uint32), np.zeros(b, np.uint32)
    path[-1, :3], accepted[-1] = [1, 2, 4], 3
    after = np.zeros(b, np.uint32)
    d_after = gpu(after)
    gpu.hip.cache_commit(gpu.dev, [dk], [dv], gpu(ctx), gpu(path), gpu(accepted), (b, t, h, hd, cap), d_after)
    ref.commit([kc], [vc], ctx[-1:], path[-1:], accepted[-1:], after[-1:])
    assert np.array_equal(gpu.back(d_after, after), after)
    cut = np.zeros(b, np.uint32)
    d_cut = gpu(cut)
    gpu.hip.cache_evict(gpu.dev, [dk], [dv], d_acc, d_after, (b, h, hd, cap), budget, recent, d_acc, d_cut)
    ref.evict([kc], [vc], acc[:, -1:], after[-1:], budget, recent, acc[:, -1:], cut[-1:], None)
    assert np.array_equal(gpu.back(d_cut, cut), cut) and np.array_equal(gpu.back(d_acc, acc), acc)
    assert np.array_equal(gpu.back(last_k, kc), kc) and np.array_equal(gpu.back(last_v, vc), vc)


def test_more_streams_than_a_grid_of_tiles(gpu):
    """2^23 + 5 streams of one row and one key, which gets the whole weight: the output follows from the value
    alone, so one row of all 256 values says what it is. As a tree and as a causal row with weights."""
    b, hd = 2 ** 23 + 5, 16
    r = np.random.default_rng(8)
    every = np.arange(-128, 128).astype(np.int8).reshape(1, 1, 16, 16)  # sixteen heads of one key
    one, out16 = np.zeros((1, 1, 16, 16), np.int8), np.zeros((1, 1, 16, 16), np.int8)
    ref.mass(one, one.reshape(1, 16, 1, 16), every.reshape(1, 16, 1, 16), np.ones(1, np.uint32), None,
             np.zeros((1, 16, 1), np.uint64), RULE, TABLE, out16)
    lut = out16.reshape(256)
    q = r.integers(-128, 128, (b, 1, 1, hd)).astype(np.int8)
    kv = r.integers(-128, 128, (b, 1, 1, hd)).astype(np.int8)
    expect = lut[kv.astype(np.int16) + 128]
    d_q, d_kv, rule, dims = gpu(q), gpu(kv), gpu.rule(RULE, TABLE), (b, 1, 1, hd, 1)
    out = np.full_like(q, 77)
    d_out = gpu(out)
    gpu.hip.attend_tree(gpu.dev, d_q, d_kv, d_kv, gpu(np.zeros(b, np.uint32)), None, gpu(np.ones(b, np.uint64)), dims, rule, d_out)
    assert np.array_equal(gpu.back(d_out, out), expect)
    d_out, d_mass = gpu(out), gpu(np.arange(b, dtype=np.uint64))
    gpu.hip.attend_mass(gpu.dev, d_q, d_kv, d_kv, gpu(np.ones(b, np.uint32)), None, d_mass, dims, rule, d_out)
    assert np.array_equal(gpu.back(d_out, out), expect)
    assert np.array_equal(gpu.back(d_mass, np.empty(b, np.uint64)), np.arange(b, dtype=np.uint64) + np.uint64(2 ** 30))


def test_more_panels_than_a_launch(gpu):
    """64 layers of 70,000 streams, more than 2^22 panels: the layers go in two launches."""
    layers, b, hd = 64, 70_000, 4
    r = np.random.default_rng(9)
    ks, vs = [[r.integers(-128, 128, (b, 1, 2, hd)).astype(np.int8) for _ in range(layers)] for _ in range(2)]
    dk, dv = [gpu(x) for x in ks], [gpu(x) for x in vs]
    dims, ones = (b, 1, hd, 2), gpu(np.ones(b, np.uint32))
    mass = r.integers(0, 3, (layers, b, 1, 2)).astype(np.uint64)
    d_mass, d_ctx, ctx = gpu(mass), gpu(np.full(b, 9, np.uint32)), np.empty(b, np.uint32)
    gpu.hip.cache_evict(gpu.dev, dk, dv, d_mass, gpu(np.full(b, 2, np.uint32)), dims, 1, 0, d_mass, d_ctx)
    second = mass[..., 1] > mass[..., 0]
    for l in range(layers):
        for x in (ks[l], vs[l]):
            x[:, :, 0][second[l]] = x[:, :, 1][second[l]]
    for d, x in zip(dk + dv, ks + vs):
        assert np.array_equal(gpu.back(d, x), x)
    mass = np.stack([mass.max(-1), np.zeros_like(mass[..., 0])], -1)
    assert np.array_equal(gpu.back(d_mass, mass), mass)
    assert (gpu.back(d_ctx, ctx) == 1).all()
    d_ctx = gpu(np.full(b, 9, np.uint32))
    gpu.hip.cache_commit(gpu.dev, dk, dv, gpu(np.zeros(b, np.uint32)), ones, ones, (b, 1, 1, hd, 2), d_ctx)
    for d, x in zip(dk + dv, ks + vs):
        x[:, :, 0] = x[:, :, 1]
        assert np.array_equal(gpu.back(d, x), x)
    assert (gpu.back(d_ctx, ctx) == 1).all()
