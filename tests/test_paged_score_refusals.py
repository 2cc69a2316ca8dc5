"""The refusals of the paged caches' entries and of the scores, without a GPU: every check comes before the device is
used, so a device that is never opened serves."""

import ctypes as C

import pytest

from taco_amd import hip

FAKE = (C.c_char * 4096)()
BASE = (C.addressof(FAKE) + 255) // 256 * 256
BAD, UNSUPPORTED = hip.HS_INVALID_ARGUMENT, hip.HS_UNSUPPORTED


class Dev:
    h = BASE


CACHE = hip.PagedCache(BASE, BASE, BASE, BASE, 10, 2, 64, 64, 64)
RULE = hip.AttentionRule(1 << 20, 36, 1, 59, BASE, 100, 24)


def refused(kind, fn, *args, **kw):
    with pytest.raises(hip.HipError) as e:
        fn(Dev, *args, **kw)
    assert e.value.status == kind and e.value.message


def append(kind=None, cache=CACHE, k=BASE, v=BASE, table=BASE, ctx=BASE, rows=BASE, dims=(2, 3, 4), headroom=20,
           ctx_out=BASE + 64, bits=16, stride=None):
    args = (cache, k, v, table, ctx, rows, dims, headroom, ctx_out, bits, stride)
    hip.pages_append(Dev, *args) if kind is None else refused(kind, hip.pages_append, *args)


def attend(kind=None, cache=CACHE, q=BASE, table=BASE, ctx=BASE, rows=BASE, dims=(2, 3, 4, 4, 200), rule=RULE, out=BASE + 2048, **kw):
    args = (cache, q, table, ctx, rows, dims, rule, out)
    hip.attend_paged(Dev, *args, **kw) if kind is None else refused(kind, hip.attend_paged, *args, **kw)


def score(kind=None, logits=BASE, tokens=BASE, table=BASE, dims=(2, 100, 50), top=3, outs=(BASE,) * 5, bits=32, stride=None):
    args = (logits, tokens, table, dims, top, *outs, bits, stride)
    hip.score_tokens(Dev, *args) if kind is None else refused(kind, hip.score_tokens, *args)


@pytest.mark.parametrize("fn", [append, attend])
def test_pools(fn):
    for name in ("k", "v", "k_scale", "v_scale"):
        fn(BAD, cache=CACHE._replace(**{name: None}))
        fn(BAD, cache=CACHE._replace(**{name: BASE + 2}))
    fn(BAD, cache=CACHE._replace(k=BASE + 8))
    for hd in (0, 8, 72, 272):
        fn(UNSUPPORTED, cache=CACHE._replace(head_dim=hd))
    for page in (0, 8, 48, 2048, 2 ** 32):
        fn(UNSUPPORTED, cache=CACHE._replace(page=page))
    for pages in (0, 2 ** 31, 2 ** 32 + 1, -1):
        fn(UNSUPPORTED, cache=CACHE._replace(pages=pages))
    for heads in (0, 65536):
        fn(UNSUPPORTED, cache=CACHE._replace(kv_heads=heads))
    for most in (0, 1025):
        fn(UNSUPPORTED, cache=CACHE._replace(max_scale=most))


def test_append_refusals():
    for name in ("k", "v", "table", "ctx"):
        append(BAD, **{name: None})
    for name in ("k", "v"):
        append(BAD, **{name: BASE + 8})
    for name in ("table", "ctx", "rows", "ctx_out"):
        append(BAD, **{name: BASE + 2})
    for bits in (0, 4, 32):
        append(UNSUPPORTED, bits=bits)
    for headroom in (0, 15, 65, -1, 2 ** 32 + 16):
        append(UNSUPPORTED, headroom=headroom)
    append(UNSUPPORTED, dims=(2, 3, 0))
    append(UNSUPPORTED, dims=(2, 3, 2 ** 25))   # 2^31 tokens of a stream
    append(UNSUPPORTED, dims=(2 ** 20, 2 ** 6, 4))
    append(UNSUPPORTED, dims=(-1, 3, 4))
    for stride in (127, 132, 2 ** 41, -128):    # 128 values a token
        append(UNSUPPORTED, stride=stride)
    append(UNSUPPORTED, bits=8, stride=136)
    append(BAD, ctx_out=BASE + 4)               # on the second count
    append(BAD, ctx=BASE + 128, ctx_out=BASE)   # on rows
    append(UNSUPPORTED, dims=(2 ** 25 - 8, 1, 4), ctx_out=BASE + 2 ** 40)    # 2^26 waves for keys and values
    append(UNSUPPORTED, dims=(2 ** 23, 3, 4), ctx_out=BASE + 2 ** 40)        # two runs of a stream
    append(dims=(0, 3, 4))
    append(dims=(2, 0, 4))


def test_attend_refusals():
    for name in ("q", "table", "ctx", "out"):
        attend(BAD, **{name: None})
    for name in ("q", "out"):
        attend(BAD, **{name: BASE + 8})
    for name in ("table", "ctx", "rows"):
        attend(BAD, **{name: BASE + 2})
    for rule in (RULE._replace(attn_exp=None), RULE._replace(attn_exp=BASE + 1)):
        attend(BAD, rule=rule)
    attend(UNSUPPORTED, dims=(2, 3, 0, 4, 200))
    attend(UNSUPPORTED, dims=(2, 3, 5, 4, 200))          # 2 heads in the cache
    attend(UNSUPPORTED, dims=(2, 3, 4, 4, 0))
    attend(UNSUPPORTED, dims=(2, 3, 4, 4, 257))          # 4 pages of 64
    attend(UNSUPPORTED, dims=(2, 3, 4, 2 ** 20, 2 ** 22 + 1))
    attend(UNSUPPORTED, dims=(2 ** 12, 2 ** 12, 4, 4, 200))
    attend(UNSUPPORTED, dims=(2, 3, 4, -1, 200))
    for stride in (240, 264, 2 ** 41, -256):
        attend(UNSUPPORTED, q_stride=stride)
    for rule in (RULE._replace(length=0), RULE._replace(length=2 ** 31), RULE._replace(score_m=0), RULE._replace(score_m=-5),
                 RULE._replace(score_m=2 ** 25), RULE._replace(softmax_p=25)):
        attend(UNSUPPORTED, rule=rule)
    attend(UNSUPPORTED, cache=CACHE._replace(max_scale=65))  # counts as 128: 2^24 128 is past 2^30
    attend(UNSUPPORTED, dims=(2 ** 21, 1, 4, 4, 200), out=BASE + 2 ** 40)    # 2^22 workgroups
    attend(BAD, workspace=BASE + 16, workspace_bytes=1 << 40)
    attend(BAD, q=BASE, out=BASE + 1024)                 # 6 rows of 256
    attend(BAD, q=BASE + 1024, out=BASE)
    attend(BAD, dims=(1, 1, 4, 4, 200), q=BASE, q_stride=4096, out=BASE + 240)
    # beside q, also in the rest of a wider row or between two: refused for its workspace, which is checked after
    for kw in (dict(dims=(1, 1, 4, 4, 200), q_stride=4096, out=BASE + 256), dict(q_stride=4096, out=BASE + 256),
               dict(q_stride=2048, out=BASE + 5 * 2048 + 256)):
        with pytest.raises(hip.HipError, match="workspace"):
            attend(workspace=BASE + 16, workspace_bytes=1 << 40, **kw)
    attend(dims=(0, 3, 4, 4, 200))
    attend(dims=(2, 0, 4, 4, 200))


def test_workspaces():
    size = hip.attend_paged_workspace
    for dims in ((0, 1, 4, 2, 64, 200), (2, 0, 4, 2, 64, 200), (2, 1, 0, 2, 64, 200), (2, 1, 4, 0, 64, 200), (2, 1, 5, 2, 64, 200),
                 (2, 1, 4, 2, 0, 200), (2, 1, 4, 2, 272, 200), (2, 1, 4, 2, 64, 0), (2, 1, 4, 2, 64, 2 ** 22 + 1),
                 (2 ** 40, 1, 4, 2, 64, 200), (2 ** 20, 2 ** 20, 4, 2, 64, 200), (2, 1, 2 ** 40, 2, 64, 200)):
        assert size(*dims) == 0, dims
    with pytest.raises(hip.Unsupported):
        size(-1, 1, 4, 2, 64, 200)


def test_score_refusals():
    score(BAD, logits=None)
    score(BAD, table=None)
    score(BAD, tokens=None)
    score(BAD, logits=BASE + 2)
    score(BAD, logits=BASE + 4, bits=64)
    score(BAD, table=BASE + 4)
    score(BAD, tokens=BASE + 1)
    for i in range(5):
        score(BAD, outs=[BASE + 2 if i == j else BASE for j in range(5)])
    for bits in (0, 16):
        score(UNSUPPORTED, bits=bits)
    for dims in ((2, 0, 50), (2, 2 ** 24, 50), (2, 2 ** 24 + 1, 50), (2, 100, 0), (2, 100, 2 ** 31), (2 ** 22, 100, 50), (-1, 100, 50)):
        score(UNSUPPORTED, dims=dims)
    for top in (65, 101, -1):
        score(UNSUPPORTED, top=top)
    score(UNSUPPORTED, dims=(2, 2, 50))  # 3 alternatives of 2 symbols
    for stride in (99, 2 ** 41, -100):
        score(UNSUPPORTED, stride=stride)
    score(dims=(0, 100, 50))


def test_tensors():
    """Tensors of other types, shapes and places are refused before their addresses are used."""
    torch = pytest.importorskip("torch")

    class Fake:
        is_cuda = True

        def __init__(self, x):
            self.x, self.shape, self.dtype = x, x.shape, x.dtype

        def __getattr__(self, name):
            return getattr(self.x, name)

        def data_ptr(self):
            return BASE

    rows = lambda dtype, *shape: Fake(torch.zeros(shape or (2, 3, 2, 64), dtype=dtype))  # noqa: E731
    good = rows(torch.int16)
    for bad in (rows(torch.float16), rows(torch.uint8), rows(torch.int16, 2, 3, 2, 32), rows(torch.int8),
                Fake(torch.zeros(2, 3, 2, 128, dtype=torch.int16)[..., ::2]), Fake(torch.zeros(2, 2, 3, 64, dtype=torch.int16).transpose(1, 2)),
                Fake(torch.zeros(2, 6, 2, 64, dtype=torch.int16)[:, :3]), torch.zeros(2, 3, 2, 64, dtype=torch.int16)):
        with pytest.raises(ValueError):
            append(k=good, v=bad, bits=None)
        with pytest.raises(ValueError):
            append(k=bad, v=good, bits=None)
    with pytest.raises(ValueError):  # keys and values at different distances
        append(k=good, v=Fake(torch.zeros(2, 3, 2, 2, 64, dtype=torch.int16)[:, :, 0]), bits=None)
    for bad in (rows(torch.int16, 2, 3, 4, 64), rows(torch.int8, 2, 3, 2, 64), torch.zeros(2, 3, 4, 64, dtype=torch.int8)):
        with pytest.raises(ValueError):
            attend(q=bad)
    for bad in (rows(torch.float32, 2, 100), rows(torch.int32, 2, 99), Fake(torch.zeros(100, 2, dtype=torch.int32).T),
                torch.zeros(2, 100, dtype=torch.int32)):
        with pytest.raises(ValueError):
            score(logits=bad, bits=None)
    kv = torch.zeros(2, 3, 2, 2, 64, dtype=torch.int16)  # parts of wider rows
    assert hip._rows_of(Fake(kv[:, :, 1]), None, None, (2, 3, 2, 64)) == (BASE, 16, 256)
    assert hip._rows_of(Fake(kv[:1, :1, 1]), None, None, (1, 1, 2, 64)) == (BASE, 16, 128)


def test_batch_tokens():
    """What run_scored makes of its tokens: other numbers than symbols and `none` stay outside the vocabulary."""
    class Batch:
        vocab = 300

    seen = []

    def call(t, *out):
        seen.extend(C.cast(t, C.POINTER(C.c_uint32))[:8])
        return 0

    out = hip.HipBatch._scored(Batch, 8, [0, -1, 299, 300, 2 ** 32 - 1, 2 ** 32, 2 ** 40, -2], 2, call)
    none = hip.HS_NO_TOKEN
    assert seen == [0, none, 299, 300, none, 300, 300, 300] and out.top_tokens.shape == (8, 2)
    with pytest.raises(hip.LengthMismatch):
        hip.HipBatch._scored(Batch, 3, [1], 2, call)
    with pytest.raises(hip.Unsupported):
        hip.HipBatch._scored(Batch, 3, [1, 2, 3], -1, call)


def test_workspaces_of_other_head_dims():
    """Head dims that the call refuses need no workspace; 1 to 3 once divided by zero."""
    for hd in (1, 2, 3, 4, 8, 15, 17, 72, 2 ** 32 + 16):
        for t, keys in ((1, 100), (1, 20_000), (20, 9000)):
            assert hip.attend_paged_workspace(1, t, 1, 1, hd, keys) == 0, hd
    assert hip.attend_paged_workspace(1, 1, 1, 1, 16, 20_000) > 0
    assert hip.attend_paged_workspace(1, 1, 65536, 65536, 16, 20_000) == 0  # heads of the cache that the call refuses


def test_batch_tokens_of_other_kinds():
    """None is no token, alone among others and for every input; whole numbers of other types are themselves; what is no whole
    number, and an array of another shape, is refused."""
    import numpy as np

    class Batch:
        vocab = 300

    def words(tokens, n):
        seen = []
        hip.HipBatch._scored(Batch, n, tokens, 0, lambda t, *out: seen.extend(C.cast(t, C.POINTER(C.c_uint32))[:n]) or 0)
        return seen

    none = hip.HS_NO_TOKEN
    assert words([7, None, 2 ** 40, -3], 4) == [7, none, 300, 300]
    assert words([None, None], 2) == [none, none]
    assert words([3.0, 4.0], 2) == [3, 4] and words([3.0, None], 2) == [3, none]
    assert words(np.array([[5], [6]]), 2) == [5, 6] and words(np.array([200, 1], np.uint8), 2) == [200, 1]
    assert words(np.array([2 ** 64 - 1, 5], np.uint64), 2) == [300, 5] and words([], 0) == []
    for bad in ([5.7, 1], [float("nan"), 1], [float("inf"), 1], [None, 0.5], ["5", "6"], [1j, 2]):
        with pytest.raises(hip.Unsupported):
            words(bad, 2)
    for bad in (np.zeros((2, 3), int), np.zeros((1, 2), int), np.zeros((2, 1, 1), int), 5, [1, 2, 3], [None]):
        with pytest.raises(hip.LengthMismatch):
            words(bad, 2)


def test_batch_alternatives():
    """More than 64 alternatives are refused before arrays of their size are made."""
    class Batch:
        vocab = 2 ** 20

    def call(*args):
        raise AssertionError("the library is called")

    for top in (65, 2 ** 31 - 1, 2 ** 31, 2 ** 70, -1):
        with pytest.raises(hip.Unsupported):
            hip.HipBatch._scored(Batch, 1, None, top, call)


def test_results_that_overlap():
    """Results that share memory, also of a few bytes, are refused; side by side, or without alternatives, they are not."""
    rows, top = 5, 3
    sizes = [4 * rows] * 3 + [4 * rows * top] * 2
    at = [BASE + sum(sizes[:i]) for i in range(5)]
    for i in range(5):
        for j in range(i):
            for x, y in ((i, j), (j, i)):
                outs = [None] * 5
                outs[x], outs[y] = BASE + 1024, BASE + 1024 + sizes[x] - 4  # y starts on the last word of x
                score(BAD, dims=(rows, 100, 50), top=top, outs=outs)
                outs[y] = BASE + 1024
                score(BAD, dims=(rows, 100, 50), top=top, outs=outs)
    # a result that lies between others; and one over alternatives of no size, refused for the number of rows only
    score(BAD, dims=(rows, 100, 50), top=top, outs=at[:4] + [at[4] - 4])
    score(dims=(0, 100, 50), top=top, outs=(BASE,) * 5)


class OnGpu:
    """A tensor as if on the GPU, whose address no call uses."""
    is_cuda = True

    def __init__(self, x):
        self.x, self.shape, self.dtype = x, x.shape, x.dtype

    def __getattr__(self, name):
        return getattr(self.x, name)


class Library:
    """Takes every call."""

    def __getattr__(self, name):
        return lambda *args: 0


def test_arrays(monkeypatch):
    """Tensors that are too short or of another type for what the call reads or writes are refused; longer ones and other
    types of the same integers are taken."""
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(hip, "lib", Library)
    cache = {"k": (torch.int8, 10 * 2 * 64 * 64), "v": (torch.int8, 10 * 2 * 64 * 64), "k_scale": (torch.int32, 20), "v_scale": (torch.int32, 20)}
    calls = [
        (append, {"table": (torch.int32, 8), "ctx": (torch.int32, 2), "rows": (torch.int32, 2), "ctx_out": (torch.int32, 2)}),
        (attend, {"table": (torch.int32, 8), "ctx": (torch.int32, 2), "rows": (torch.int32, 2), "out": (torch.int8, 6 * 256)}),
        (score, {"tokens": (torch.int32, 2), "table": (torch.int64, 50)}),
    ]
    other = {torch.int8: (torch.int16, torch.float16), torch.int32: (torch.int64, torch.float32, torch.int16), torch.int64: (torch.int32, torch.float64),
             torch.float32: (torch.float64, torch.int32, torch.bfloat16)}
    same = {torch.int8: torch.uint8, torch.int32: torch.uint32, torch.int64: torch.uint64, torch.float32: torch.float32}

    def each(give, dtype, n):
        give(OnGpu(torch.zeros(n, dtype=dtype)))
        give(OnGpu(torch.zeros(n + 3, dtype=same[dtype])))
        for bad in [torch.zeros(n - 1, dtype=dtype), torch.zeros(2 * n, dtype=dtype)[::2]] + [torch.zeros(n, dtype=d) for d in other[dtype]]:
            with pytest.raises(ValueError):
                give(OnGpu(bad))
        with pytest.raises(ValueError):
            give(torch.zeros(n, dtype=dtype))  # in host memory

    for fn, arrays in calls:
        for name, (dtype, n) in arrays.items():
            each(lambda x: fn(**{name: x}), dtype, n)
    for fn in (append, attend):
        for name, (dtype, n) in cache.items():
            each(lambda x: fn(cache=CACHE._replace(**{name: x})), dtype, n)
    each(lambda x: attend(rule=RULE._replace(attn_exp=x)), torch.int32, 100)
    for i, (dtype, n) in enumerate([(torch.float32, 2), (torch.int32, 2), (torch.float32, 2), (torch.int32, 6), (torch.float32, 6)]):
        each(lambda x: score(outs=[x if i == j else BASE for j in range(5)]), dtype, n)
    space = OnGpu(torch.zeros(100, dtype=torch.int32))
    attend(workspace=space, workspace_bytes=400)
    with pytest.raises(ValueError):
        attend(workspace=space, workspace_bytes=401)
