"""Scores of rows of logits against the 64-bit forms of paged_ref.py: ranks and alternatives for equality, logarithms
within the header's bounds; rows of both types, odd vocabularies and strides, ties, tables of every length, weights of 0; and
through the batch against the weights that run_weights gives.

Tolerances: a log probability is rounded to 32 bits once from a 64-bit value whose error is some 2^-50 of it: half a unit in the last
place, so 1 here. The entropy may be 2^-20 of itself off (8 units of 2^-23)."""

import numpy as np
import pytest

from oracle import oracle as O
from taco_amd import synth
from tests import paged_ref as ref
from tests.test_gpu_tree_cache import Gpu

pytestmark = pytest.mark.gpu

WEIGHTS = np.rint(2.0 ** 40 * np.exp(-np.arange(8192) / 256)).astype(np.uint64)


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


def check(gpu, logits, table, tokens, top, pad=0):
    rows, vocab = logits.shape
    print(f"score {rows}x{vocab} {logits.dtype} table {len(table)} top {top}", flush=True)
    wide = np.full((rows, vocab + pad), np.iinfo(logits.dtype).max, logits.dtype)
    wide[:, :vocab] = logits
    t = None if tokens is None else np.asarray(tokens, np.uint32)
    outs = [np.full(rows, 7, np.float32), np.full(rows, 7, np.uint32), np.full(rows, 7, np.float32),
            np.full((rows, top), 7, np.uint32), np.full((rows, top), 7, np.float32)]
    held = [gpu(x) for x in outs]
    args = held if t is not None else [None, None] + held[2:]
    gpu.hip.score_tokens(gpu.dev, gpu(wide), None if t is None else gpu(t), gpu(table), (rows, vocab, len(table)), top, *args,
                         bits=8 * logits.dtype.itemsize, stride=vocab + pad)
    got = [gpu.back(p, x) for p, x in zip(held, outs)]
    lp, rank, entropy, tops, tops_lp = ref.scores(logits, table, t, top)
    if t is not None:
        assert np.array_equal(got[1], rank)
        ref.close(got[0], lp, 1)
    assert np.array_equal(got[3], tops), np.argwhere(got[3] != tops)[:5]
    ref.close(got[4], tops_lp, 1)
    ref.close(got[2], entropy, 8)


def normal(r, rows, vocab, dtype, std=700.0, mean=0):
    return (np.rint(r.standard_normal((rows, vocab)) * std) + mean).astype(dtype)


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
@pytest.mark.parametrize("rows,vocab,top,pad", [
    (1, 1, 1, 0), (1, 2, 0, 0), (3, 63, 5, 1), (2, 64, 64, 0), (5, 299, 16, 3), (2, 4096, 1, 0), (3, 4097, 7, 2), (2, 50257, 8, 0),
    (1, 50257, 64, 7), (2, 70001, 5, 0), (1, 150_000, 33, 1)])
def test_shapes(gpu, rows, vocab, top, pad, dtype):
    r = np.random.default_rng(vocab)
    check(gpu, normal(r, rows, vocab, dtype, mean=5000), WEIGHTS, r.integers(0, vocab, rows), top, pad)


@pytest.mark.parametrize("length", [1, 2, 64, 301, 8191, 16384, 16385, 40_000])
def test_tables(gpu, length):
    r = np.random.default_rng(length)
    table = np.rint(2.0 ** 40 * np.exp(-np.arange(length) / max(1, length / 30))).astype(np.uint64)
    logits = normal(r, 4, 3001, np.int64, std=length / 6 + 1)
    check(gpu, logits, table, logits.argmax(axis=1), 10)


def test_ties(gpu):
    """All equal, two values, ties of more symbols than are asked for, and the largest at the end."""
    for vocab in (500, 9000, 50257):
        logits = np.zeros((5, vocab), np.int32)
        logits[1, 100::2] = -3
        logits[2] = np.arange(vocab) % 7
        logits[3, -1] = 1
        logits[4] = -(np.arange(vocab) // 600)
        check(gpu, logits, WEIGHTS, [0, vocab - 1, 77, vocab - 2, vocab // 2], 64)


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
@pytest.mark.parametrize("vocab,pad", [(53_250, 0), (99_999, 1), (135_165, 2), (135_172, 0)])
def test_long_rows(gpu, vocab, pad, dtype):
    """Rows whose symbols are held in 16 bits each, relative to the largest of the first ones: further ones far above it,
    by as much as that holds and by more, the least numbers there are, and the largest as the last."""
    r = np.random.default_rng(vocab)
    low = np.iinfo(np.int32).min
    logits = normal(r, 9, vocab, np.int64)
    logits[1, vocab - 1] = 20_000
    logits[2, 40_000:] += 40_000
    top = logits[3, :16_384].max()                      # (the first groups are at least these symbols' part)
    logits[3, 50_000] = top + 65_535 - len(WEIGHTS) - 63
    logits[4, 50_000:50_010] = 70_000 + np.arange(10)   # past it
    logits[5] += low + 4000                             # the table reaches below the least number
    logits[5] = np.maximum(logits[5], low)
    logits[6] = low
    logits[6, 52_000] = low + 100
    logits[7] = r.integers(low, -low, vocab)
    logits[8, ::3] = low
    check(gpu, logits.astype(dtype), WEIGHTS, r.integers(0, vocab, 9), 8, pad)
    check(gpu, logits.astype(dtype), WEIGHTS[:16], None, 1, pad)


def test_more_ties_than_a_list(gpu):
    """Thousands of equal symbols at the border of the alternatives, some before them, and past the table's end; the token
    one of them."""
    r = np.random.default_rng(12)
    for vocab in (700, 5000, 50257, 120_000):
        logits = np.full((6, vocab), -700, np.int32)
        logits[0, r.integers(0, vocab, 20)] = r.integers(0, 300, 20)
        logits[1, :] = -9000
        logits[1, vocab - 5:] = np.arange(5)
        logits[2, : vocab // 2] = -20_000
        logits[2, vocab // 2] = 0
        logits[3, r.random(vocab) < 0.5] = -701
        logits[4, -1] = 5
        logits[5] = r.integers(-100_000, 0, vocab)
        for dtype in (np.int32, np.int64):
            check(gpu, logits.astype(dtype), WEIGHTS, r.integers(0, vocab, 6), 64)


def test_weights_of_zero(gpu):
    """A table that ends in zeros: alternatives and tokens without weight have log probability minus infinity."""
    r = np.random.default_rng(2)
    table = WEIGHTS[:300].copy()
    table[20:] = 0
    logits = normal(r, 6, 2000, np.int64, std=100)
    check(gpu, logits, table, [int(x) for x in logits.argmin(axis=1)], 30)
    check(gpu, logits, np.zeros(10, np.uint64), [0] * 6, 3)


def test_certain_rows(gpu):
    """One symbol far above the others: probabilities within 2^-30 of 1 and entropies of that size keep their digits."""
    logits = np.full((4, 1000), -5000, np.int64)
    for i, lead in enumerate((0, 3000, 5200, 6500)):
        logits[i, 17] = -5000 + lead
    check(gpu, logits, WEIGHTS, [17] * 4, 3)


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
def test_far_logits(gpu, dtype):
    """Distances that pass 32 bits (and 63), and the types' ends."""
    r = np.random.default_rng(4)
    info = np.iinfo(dtype)
    logits = normal(r, 4, 700, dtype)
    logits[1, 300:] = info.min
    logits[2, 5] = info.max
    logits[2, 6] = info.max - 100
    logits[2, 7] = info.min
    logits[3] = r.integers(info.min, info.max, 700, dtype)
    check(gpu, logits, WEIGHTS, [5, 300, 6, 0], 20)


def test_rows_without_tokens(gpu):
    r = np.random.default_rng(5)
    logits = normal(r, 6, 1234, np.int32)
    check(gpu, logits, WEIGHTS, None, 4)
    check(gpu, logits, WEIGHTS, [0, 0xFFFFFFFF, 1234, 1233, 5, 0x80000000], 4)


def test_only_what_is_asked_for(gpu):
    """Results that are NULL are left out, the others stay as they are."""
    r = np.random.default_rng(6)
    logits, tokens = normal(r, 3, 5000, np.int32), np.array([1, 2, 3], np.uint32)
    lp, rank, entropy, tops, tops_lp = ref.scores(logits, WEIGHTS, tokens, 4)
    for keep in range(5):
        outs = [np.zeros(3, np.float32), np.zeros(3, np.uint32), np.zeros(3, np.float32), np.zeros((3, 4), np.uint32),
                np.zeros((3, 4), np.float32)]
        held = gpu(outs[keep])
        gpu.hip.score_tokens(gpu.dev, gpu(logits), gpu(tokens), gpu(WEIGHTS), (3, 5000, 8192), 4,
                             *[held if i == keep else None for i in range(5)], bits=32)
        got = gpu.back(held, outs[keep])
        if keep in (1, 3):
            assert np.array_equal(got, (lp, rank, entropy, tops, tops_lp)[keep])
        else:
            ref.close(got, (lp, rank, entropy, tops, tops_lp)[keep], 8)


def test_many_rows(gpu):
    r = np.random.default_rng(7)
    check(gpu, normal(r, 3001, 299, np.int64, std=60), WEIGHTS[:301], r.integers(0, 299, 3001), 5)
    check(gpu, normal(r, 300, 4000, np.int32), WEIGHTS, r.integers(0, 4000, 300), 2)


# ---- Through the batch ---------------------------------------------------------------------------


def want_of(w, token, top):
    """The scores of a row of weights: the order by distance is that by weight while weights differ, as those of 256 and
    more do (the tables step by a 256th)."""
    return ref.scores_of(w, -w.astype(np.int64), token, top)


def likely(r, weights):
    """A token of each row that the order by weight places."""
    return [int(r.choice(np.nonzero(w >= 1024)[0])) for w in weights]


def check_scores(got, weights, tokens, top):
    for i, w in enumerate(weights):
        lp, rank, entropy, tops, tops_lp = want_of(w, None if tokens is None else int(tokens[i]), top)
        if tokens is not None:
            assert got.rank[i] == rank, i
            ref.close(got.logprob[i:i + 1], np.array([lp]), 1)
        ref.close(got.entropy[i:i + 1], np.array([entropy]), 8)
        assert np.array_equal(got.top_tokens[i], tops), i
        ref.close(got.top_logprob[i], tops_lp, 1)


MODELS = {"tiny": lambda: O.build_model(O.tiny_dims(), 0x7AC0_0001, 64),
          "heads32": lambda: synth.build_model(synth.Dims(1, 2, 64, 128))}


@pytest.fixture(scope="module")
def dev():
    from taco_amd import hip
    return hip.HipDevice.open(0)


@pytest.mark.parametrize("name", ["tiny", "heads32"])
def test_batch_scores(dev, name):
    """run_scored gives the scores of the weights that run_weights gives, over several slots, passes and a restart; and
    positions move as they do there."""
    from taco_amd import hip
    model = hip.HipModel.load(dev, MODELS[name]())
    r, V, C = np.random.default_rng(1), model.vocab_size(), model.n_ctx()
    n = min(C + 5, 80)
    inputs = [(s, int(x)) for s in range(3) for x in r.integers(0, V - 1, n)]
    plain, scored = (hip.HipBatch(model, 3, 64) for _ in range(2))
    weights = plain.run_weights(inputs)
    tokens = likely(r, weights)
    tokens[5] = -1
    got = scored.run_scored(inputs, tokens, 6)
    tokens[5] = 0xFFFFFFFF
    check_scores(got, weights, tokens, 6)
    assert got.logprob[5] == 0 and got.rank[5] == hip.HS_NO_TOKEN
    assert [plain.position(s) for s in range(3)] == [scored.position(s) for s in range(3)]
    got = scored.run_scored([(1, 3)], None, 20)
    assert got.logprob is None and got.rank is None
    check_scores(got, plain.run_weights([(1, 3)]), None, 20)
    assert scored.run_scored([], None, 3).top_tokens.shape == (0, 3)


def test_tree_scores(dev):
    """A tree grown by the alternatives: each node's scores are those of its weights, and no position moves."""
    from taco_amd import hip
    model = hip.HipModel.load(dev, MODELS["tiny"]())
    batch = hip.HipBatch(model, 2, 64)
    batch.run_without_readback([(s, 5 + s) for s in range(2)])
    first = batch.run_scored([(0, 7), (1, 8)], None, 3)
    inputs = [(s, int(t)) for s in range(2) for t in first.top_tokens[s]]
    parents = [-1] * 6
    inputs += [(0, 1), (1, 2)]
    parents += [1, 5]
    weights = batch.run_tree_weights(inputs, parents)
    tokens = likely(np.random.default_rng(2), weights)
    tokens[7] = hip.HS_NO_TOKEN
    check_scores(batch.run_tree_scored(inputs, parents, tokens, 4), weights, tokens, 4)
    assert [batch.position(s) for s in range(2)] == [2, 2]
    batch.commit_paths({0: [1, 3], 1: []})
    assert [batch.position(s) for s in range(2)] == [4, 2]


def test_wide_models_and_long_tables(dev):
    """The i64 logits of a model whose table is longer than the compact form takes, and a version-2 model."""
    from taco_amd import hip
    r = np.random.default_rng(3)
    for kw in ({"table_len": 20_000}, {"wide": True}):
        model = hip.HipModel.load(dev, synth.build_model(synth.Dims(1, 2, 64, 128), **kw))
        V = model.vocab_size()
        inputs = [(s, int(x)) for s in range(2) for x in r.integers(0, V, 9)]
        plain, scored = (hip.HipBatch(model, 2, 32) for _ in range(2))
        weights = plain.run_weights(inputs)
        tokens = likely(r, weights)
        check_scores(scored.run_scored(inputs, tokens, 5), weights, tokens, 5)


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
@pytest.mark.parametrize("vocab", [1021, 1022, 16381, 16382, 53245, 53246, 131_072])
def test_around_the_forms(gpu, vocab, dtype):
    """Vocabularies at the ends of what a wave's and a workgroup's registers hold, every alignment of a row, and ties."""
    r = np.random.default_rng(vocab)
    logits = normal(r, 4, vocab, dtype, std=300)
    logits[1, vocab // 3::5] = logits[1].max()
    check(gpu, logits, WEIGHTS, [vocab - 1, vocab - 2, 0, int(logits[3].argmax())], 9, 1)


def test_rows_that_do_not_start_at_16_bytes(gpu):
    r = np.random.default_rng(8)
    for dtype in (np.int32, np.int64):
        logits, tokens = normal(r, 3, 501, dtype), np.array([0, 250, 500], np.uint32)
        size = dtype().itemsize
        for skip in range(1, 16 // size):
            flat = np.concatenate([np.full(skip, np.iinfo(dtype).max, dtype), logits.ravel()])
            outs = [np.zeros(3, np.float32), np.zeros(3, np.uint32), np.zeros(3, np.float32)]
            held = [gpu(x) for x in outs]
            gpu.hip.score_tokens(gpu.dev, gpu(flat).value + skip * size, gpu(tokens), gpu(WEIGHTS), (3, 501, 8192), 0, *held, None, None,
                                 bits=8 * size)
            got = [gpu.back(p, x) for p, x in zip(held, outs)]
            lp, rank, entropy, _, _ = ref.scores(logits, WEIGHTS, tokens, 0)
            assert np.array_equal(got[1], rank)
            ref.close(got[0], lp, 1)
            ref.close(got[2], entropy, 8)
