"""Paged caches against the plain 64-bit forms of paged_ref.py, value for value: appended rows of both types,
chunkings, ragged counts, holes and full tables; attention of one row and of chunks, shared heads, page sizes
around the tiles, rows that see nothing, every shape of rule; the other attention operators' results where the
scales are 1; and a serving loop of both with the scores."""

import ctypes as C

import numpy as np
import pytest

from tests import paged_ref as ref
from tests.test_gpu_tree_cache import TABLE, Gpu

pytestmark = pytest.mark.gpu

RULE = (33_000_000, 35, 1_300_000_000, 56, 24)  # scales up to 64


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


def tables(r, b, width, pages, holes=0.0):
    t = r.permutation(pages)[:b * width].reshape(b, width).astype(np.uint32)
    t[r.random(t.shape) < holes] = np.uint32(2 ** 32 - 1)
    return t


def device_cache(gpu, pool):
    held = [gpu(x) for x in pool.arrays()]
    pages, kv_heads, page, hd = pool.shape
    return gpu.hip.PagedCache(*held, pages, kv_heads, page, hd, pool.max_scale)


def check_pool(gpu, cache, pool):
    for name, got, want in zip(("k", "v", "k_scale", "v_scale"), cache[:4], pool.arrays()):
        assert np.array_equal(gpu.back(got, want), want), name


def new_rows(r, b, t, kvh, hd, bits, big=2000):
    dtype, most = (np.int8, 128) if bits == 8 else (np.int16, big)
    return [r.integers(-most, most, (b, t, kvh, hd)).astype(dtype) for _ in range(2)]


def run_append(gpu, cache, k, v, table, ctx, rows, headroom=20, ctx_out=None):
    b, t, kvh, hd = k.shape
    gpu.hip.pages_append(gpu.dev, cache, gpu(k), gpu(v), gpu(table), gpu(ctx), None if rows is None else gpu(rows),
                         (b, t, table.shape[1]), headroom, ctx_out, bits=8 * k.dtype.itemsize)


@pytest.mark.parametrize("b,t,kvh,hd,page,width,ctx,rows,bits,max_scale", [
    (1, 1, 1, 16, 16, 1, [0], None, 16, 64),
    (5, 1, 12, 64, 64, 4, [0, 63, 64, 100, 255], None, 16, 64),
    (5, 1, 12, 64, 64, 4, [0, 63, 64, 100, 256], None, 8, 1),       # the last stream is full
    (3, 37, 4, 80, 16, 5, [0, 7, 60], [37, 0, 36], 16, 1024),       # the last one runs over
    (3, 37, 4, 80, 16, 5, [0, 7, 1 << 31], [37, 5, 1 << 31], 8, 7),
    (2, 130, 3, 256, 32, 9, [31, 32], None, 16, 64),
    (2, 200, 25, 64, 128, 3, [127, 1], [200, 129], 16, 100),
    (1, 1100, 2, 32, 1024, 2, [900], None, 16, 64),
    (70, 3, 1, 48, 16, 2, [14], None, 16, 64)])
def test_append(gpu, b, t, kvh, hd, page, width, ctx, rows, bits, max_scale):
    print(f"append {b}x{t}x{kvh}x{hd} page {page}", flush=True)
    r = np.random.default_rng(b + t)
    pool = ref.Pool(r, b * width + 3, kvh, page, hd, max_scale)
    cache, table = device_cache(gpu, pool), tables(r, b, width, b * width + 3, 0.1 if b > 2 else 0)
    ctx = np.resize(np.array(ctx, np.uint32), b)
    rows = None if rows is None else np.resize(np.array(rows, np.uint32), b)
    k, v = new_rows(r, b, t, kvh, hd, bits)
    out = np.zeros(b, np.uint32)
    d_out = gpu(out)
    run_append(gpu, cache, k, v, table, ctx, rows, 20, d_out)
    want = out.copy()
    ref.append(pool, k, v, table, ctx, rows, 20, want)
    check_pool(gpu, cache, pool)
    assert np.array_equal(gpu.back(d_out, out), want)


@pytest.mark.parametrize("headroom", [16, 64])
def test_append_extremes(gpu, headroom):
    """Rows of zeros, of the types' ends, of one large value after a small first row (it saturates), and the halves
    between two stored values."""
    r = np.random.default_rng(1)
    pool = ref.Pool(r, 6, 2, 16, 64, 1024)
    cache, table = device_cache(gpu, pool), np.arange(6, dtype=np.uint32).reshape(1, 6)
    k, v = (np.zeros((1, 96, 2, 64), np.int16) for _ in range(2))
    k[0, 1:20] = np.arange(-9, 10)[:, None, None]
    k[0, 20:40] = -32768
    k[0, 40:50] = 32767
    k[0, 48, 0, 3] = -32768
    k[0, 64] = 127 * 16 // headroom  # scale 1
    k[0, 65:80] = np.arange(-300, 300, 40)[:, None, None]
    k[0, 80] = 254 * 16 // headroom  # scale 2: odd values are halves
    k[0, 81:96] = np.arange(-7, 8)[:, None, None]
    v[:] = k[:, ::-1]
    run_append(gpu, cache, k, v, table, np.zeros(1, np.uint32), None, headroom)
    ref.append(pool, k, v, table, np.zeros(1), None, headroom)
    check_pool(gpu, cache, pool)


def test_append_is_the_same_in_any_chunks(gpu):
    r = np.random.default_rng(3)
    k, v = new_rows(r, 2, 150, 3, 64, 16)
    table, pools = tables(r, 2, 5, 10), []
    for chunks in ([150], [1] * 150, [15, 17, 16, 1, 63, 38]):
        pool = ref.Pool(np.random.default_rng(4), 10, 3, 32, 64, 64)
        cache, at = device_cache(gpu, pool), 0
        for n in chunks:
            run_append(gpu, cache, k[:, at:at + n], v[:, at:at + n], table, np.full(2, at, np.uint32), None)
            at += n
        pools.append([gpu.back(x, y) for x, y in zip(cache[:4], pool.arrays())])
    for other in pools[1:]:
        for x, y in zip(pools[0], other):
            assert np.array_equal(x, y)


def check_attend(gpu, b, t, heads, kvh, hd, page, keys, ctx, rows=None, rule=RULE, exp=TABLE, max_scale=64, holes=0.0,
                 seed=1, most=128, **kw):
    print(f"attend {b}x{t}x{heads}/{kvh}x{hd} page {page} keys {keys}", flush=True)
    r = np.random.default_rng(seed)
    width = -(-keys // page) + seed % 2
    pool = ref.Pool(r, b * width + 2, kvh, page, hd, max_scale)
    pool.ks[0] = 0          # counts as 1
    pool.vs[1] = 1 << 30    # counts as max_scale
    cache, table = device_cache(gpu, pool), tables(r, b, width, b * width + 2, holes)
    q = r.integers(-most, most, (b, t, heads, hd)).astype(np.int8)
    ctx = np.resize(np.array(ctx, np.uint32), b)
    rows = None if rows is None else np.resize(np.array(rows, np.uint32), b)
    out = np.full((b, t, heads, hd), 77, np.int8)
    d_out = gpu(out)
    gpu.hip.attend_paged(gpu.dev, cache, gpu(q), gpu(table), gpu(ctx), None if rows is None else gpu(rows),
                         (b, t, heads, width, keys), gpu.rule(rule, exp), d_out, **kw)
    got = gpu.back(d_out, out)
    want = ref.attend(pool, q, table, ctx, rows, keys, rule, exp, out)
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
    check_pool(gpu, cache, pool)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("keys,ctx", [(1, [1, 0]), (64, [64, 63, 17]), (200, [200, 129, 0, 1]), (1025, [1025, 1024, 300])])
def test_one_row(gpu, page, keys, ctx):
    check_attend(gpu, len(ctx), 1, 3, 3, 64, page, keys, ctx)


@pytest.mark.parametrize("hd", [16, 32, 48, 64, 80, 112, 128, 144, 192, 256])
def test_head_dims(gpu, hd):
    check_attend(gpu, 2, 1, 2, 2, hd, 32, 300, [300, 77])
    check_attend(gpu, 2, 1, 10, 2, hd, 32, 300, [300, 77], seed=2)
    check_attend(gpu, 2, 19, 2, 2, hd, 32, 300, [300, 19], seed=3)


@pytest.mark.parametrize("heads,kvh", [(2, 1), (4, 1), (6, 2), (8, 1), (16, 1), (34, 2), (25, 25)])
def test_shared_heads(gpu, heads, kvh):
    check_attend(gpu, 3, 1, heads, kvh, 64, 64, 500, [500, 64, 3])
    check_attend(gpu, 2, 5, heads, kvh, 64, 16, 200, [200, 4], seed=2)


@pytest.mark.parametrize("t,rows", [(2, None), (4, [4, 1, 0]), (16, None), (17, [17, 16, 3]), (64, [64, 33, 0]), (100, None)])
def test_chunks(gpu, t, rows):
    """Causal chunks; the last stream's context is shorter than its rows, so that the first of them see nothing."""
    check_attend(gpu, 3, t, 4, 2, 64, 64, 400, [400, 200, t // 2], rows)


@pytest.mark.parametrize("t,heads,kvh", [(1, 2, 2), (1, 6, 1), (40, 2, 1)])
@pytest.mark.parametrize("keys", [2000, 2100, 4200, 9000, 20000])
def test_long_caches(gpu, keys, t, heads, kvh):
    check_attend(gpu, 2, t, heads, kvh, 64, 128, keys, [keys, keys // 3], seed=keys)


@pytest.mark.parametrize("keys,heads,hd", [(9000, 2, 64), (16384, 6, 64), (16385, 2, 64), (12000, 8, 48)])
def test_many_long_caches(gpu, keys, heads, hd):
    """128 panels of a few rows: those of up to 16,384 keys in one launch."""
    ctx = np.concatenate([[keys, keys - 1, 0, 1, 8192, 8193], np.linspace(3, keys, 58)]).astype(np.uint32)
    check_attend(gpu, 64, 1, heads, 2, hd, 64, keys, ctx, holes=0.05, seed=keys)


@pytest.mark.parametrize("t,heads", [(1, 2), (1, 12), (40, 2)])
def test_long_caches_with_wide_scores(gpu, t, heads):
    """A shift below 32: scores of 64 bits."""
    check_attend(gpu, 2, t, heads, 2, 64, 64, 9000, [9000, 8192], rule=(33_000_000, 20, 1_300_000_000, 56, 24), holes=0.1)
    check_attend(gpu, 64, 1, 2, 2, 64, 64, 9000, [9000, 8192, 5, 100], rule=(33_000_000, 20, 1_300_000_000, 56, 24))


@pytest.mark.parametrize("hd", [64, 112, 256])
@pytest.mark.parametrize("keys", [70, 1000, 2049, 4096, 4097])
def test_five_to_eight_rows(gpu, hd, keys):
    """Two groups of keys share an accumulator."""
    check_attend(gpu, 3, 1, 16, 2, hd, 64, keys, [keys, keys // 2, 3], holes=0.1, seed=keys)
    check_attend(gpu, 3, 5, 2, 2, hd, 16, keys, [keys, keys - 3, 3], [5, 4, 5], seed=hd)
    check_attend(gpu, 2, 3, 4, 2, hd, 32, keys, [keys, 2], rule=(33_000_000, 20, 1_300_000_000, 56, 24), exp=np.resize(TABLE, 20_000))
    check_attend(gpu, 2, 7, 2, 2, hd, 32, keys, [keys, 7], [7, 0])


@pytest.mark.parametrize("hd", [128, 256])
def test_long_caches_of_wide_heads(gpu, hd):
    for t in (1, 20):
        check_attend(gpu, 2, t, 4, 2, hd, 16, 6000, [6000, 2047], seed=t)


def test_holes(gpu):
    """Pages that are not there, whole streams of them among these."""
    for keys in (300, 5000):
        for t in (1, 20):
            check_attend(gpu, 3, t, 4, 2, 64, 16, keys, [keys, 200, 30], holes=0.5, seed=keys + t)
            check_attend(gpu, 1, t, 4, 2, 64, 16, keys, [keys], holes=1.0)


@pytest.mark.parametrize("rule", [
    (1, 0, 1, 0, 24), (33_000_000, 20, 1_300_000_000, 56, 24), (33_000_000, 31, 1_300_000_000, 56, 24),
    (33_000_000, 32, -1_300_000_000, 56, 24), (33_000_000, 60, 1, 30, 24), (33_000_000, 61, 1, 30, 24),
    (33_000_000, 200, 2 ** 31 - 1, 95, 24), (33_000_000, 35, -2 ** 31, 96, 24), (33_000_000, 35, 1_300_000_000, 32, 0),
    (33_554_431, 36, 2 ** 31 - 1, 48, 24)])
def test_rules(gpu, rule):
    for t in (1, 18):
        check_attend(gpu, 2, t, 2, 2, 64, 32, 300, [300, 20], rule=rule)
        check_attend(gpu, 1, t, 2, 2, 64, 32, 2500, [2500], rule=rule)


@pytest.mark.parametrize("exp", [np.array([5], np.int32), np.zeros(300, np.int32), np.resize(TABLE, 20_000),
                                 np.full(100, 2 ** 31 - 1, np.int32), TABLE[:257]], ids=["one", "zeros", "long", "flat", "257"])
def test_exponent_tables(gpu, exp):
    for t in (1, 18):
        check_attend(gpu, 2, t, 2, 2, 64, 32, 300, [300, 20], exp=exp)
        check_attend(gpu, 1, t, 2, 2, 64, 32, 2500, [2500], exp=exp)


@pytest.mark.parametrize("max_scale,m,p", [(1, 2 ** 31 - 1, 30), (1024, 2_097_151, 20), (3, 700_000_000, 28)])
def test_scale_limits(gpu, max_scale, m, p):
    for t in (1, 18):
        check_attend(gpu, 2, t, 2, 2, 256, 32, 300, [300, 20], rule=(m, 40, 1_300_000_000, 59, p), max_scale=max_scale)


@pytest.mark.parametrize("t", [1, 24])
def test_scales_of_one_are_the_other_rule(gpu, t):
    """The results of attend_mass on the same keys."""
    r = np.random.default_rng(9)
    b, h, hd, page, width = 2, 3, 64, 64, 8
    pool = ref.Pool(r, b * width, h, page, hd, 1)
    cache, table = device_cache(gpu, pool), tables(r, b, width, b * width)
    dense = [np.ascontiguousarray(x[table].transpose(0, 2, 1, 3, 4)).reshape(b, h, width * page, hd) for x in (pool.k, pool.v)]
    q, ctx = r.integers(-128, 128, (b, t, h, hd)).astype(np.int8), np.array([512, 100], np.uint32)
    rule = gpu.rule((1_400_000_000, 36, 1_300_000_000, 59, 30), TABLE)
    out = [gpu(np.zeros(q.shape, np.int8)) for _ in range(2)]
    gpu.hip.attend_paged(gpu.dev, cache, gpu(q), gpu(table), gpu(ctx), None, (b, t, h, width, 512), rule, out[0])
    gpu.hip.attend_mass(gpu.dev, gpu(q), gpu(dense[0]), gpu(dense[1]), gpu(ctx), None, gpu(np.zeros((b, h, 512), np.uint64)),
                        (b, t, h, hd, 512), rule, out[1])
    assert np.array_equal(*[gpu.back(x, q) for x in out])


def test_strides(gpu):
    """q, k and v as parts of wider rows."""
    r = np.random.default_rng(5)
    b, t, h, hd, page, width = 2, 6, 4, 64, 16, 4
    pool = ref.Pool(r, b * width, h, page, hd, 64)
    cache, table = device_cache(gpu, pool), tables(r, b, width, b * width)
    kv = r.integers(-3000, 3000, (b, t, 2, h, hd)).astype(np.int16)
    base, ctx, after = gpu(kv).value, np.array([0, 40], np.uint32), gpu(np.zeros(b, np.uint32))
    d_table = gpu(table)
    gpu.hip.pages_append(gpu.dev, cache, base, base + 2 * h * hd, d_table, gpu(ctx), None, (b, t, width), 20, after, bits=16,
                         stride=2 * h * hd)
    counts = np.zeros(b, np.uint32)
    ref.append(pool, kv[:, :, 0], kv[:, :, 1], table, ctx, None, 20, counts)
    check_pool(gpu, cache, pool)
    wide = r.integers(-128, 128, (b, t, 3 * h * hd + 16)).astype(np.int8)
    out = np.zeros((b, t, h, hd), np.int8)
    d_out = gpu(out)
    gpu.hip.attend_paged(gpu.dev, cache, gpu(wide).value + h * hd, d_table, after, None, (b, t, h, width, 64), gpu.rule(RULE, TABLE),
                         d_out, q_stride=3 * h * hd + 16)
    q = wide[:, :, h * hd:2 * h * hd].reshape(b, t, h, hd)
    assert np.array_equal(gpu.back(d_out, out), ref.attend(pool, q, table, counts, None, 64, RULE, TABLE, out))


def test_serving_loop(gpu):
    """A prompt in a chunk and then token by token, two layers: append, attend, and the token that the scores of the
    outputs name first becomes the next row; as the plain forms do it."""
    r = np.random.default_rng(11)
    b, h, hd, page, width, vocab = 3, 2, 64, 16, 6, 97
    pools = [ref.Pool(r, b * width, h, page, hd, 64) for _ in range(2)]
    caches, table = [device_cache(gpu, p) for p in pools], tables(r, b, width, b * width)
    embed = r.integers(-1500, 1500, (2, vocab, 3, h, hd)).astype(np.int16)  # a token's q, k and v in each layer
    head = r.integers(-40, 40, (vocab, h * hd))
    weights = np.rint(2.0 ** 40 * np.exp(-np.arange(4096) / 256)).astype(np.uint64)
    d_table, d_weights, rule = gpu(table), gpu(weights), gpu.rule(RULE, TABLE)
    ctx, tokens = np.zeros(b, np.uint32), r.integers(0, vocab, (b, 21))
    d_ctx = [gpu(ctx), gpu(ctx)]
    for step in range(30):
        t = tokens.shape[1]
        counts = ctx.copy()
        state = np.zeros((b, t, h * hd), np.int64)
        for layer in range(2):
            rows = embed[layer][tokens]
            q = np.clip(rows[:, :, 0] // 12 + state.reshape(b, t, h, hd), -128, 127).astype(np.int8)
            k, v = (np.ascontiguousarray(rows[:, :, i]) for i in (1, 2))
            gpu.hip.pages_append(gpu.dev, caches[layer], gpu(k), gpu(v), d_table, d_ctx[0], None, (b, t, width), 20, d_ctx[1], bits=16)
            ref.append(pools[layer], k, v, table, ctx, None, 20, counts)
            out = np.zeros((b, t, h, hd), np.int8)
            d_out = gpu(out)
            gpu.hip.attend_paged(gpu.dev, caches[layer], gpu(q), d_table, d_ctx[1], None, (b, t, h, width, width * page), rule, d_out)
            got = gpu.back(d_out, out)
            assert np.array_equal(got, ref.attend(pools[layer], q, table, counts, None, width * page, RULE, TABLE, out)), (step, layer)
            state = got.reshape(b, t, h * hd).astype(np.int64)
        logits = np.ascontiguousarray(state[:, -1] @ head.T)
        top = gpu(np.zeros((b, 3), np.uint32))
        gpu.hip.score_tokens(gpu.dev, gpu(logits), None, d_weights, (b, vocab, len(weights)), 3, None, None, None, top, None, bits=64)
        top = gpu.back(top, np.zeros((b, 3), np.uint32))
        assert np.array_equal(top, ref.scores(logits, weights, None, 3)[3]), step
        tokens, ctx = top[:, :1].astype(np.int64), counts
        d_ctx = d_ctx[::-1]
