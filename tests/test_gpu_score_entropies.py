"""Entropies of rows of logits within the header's bound, 2^-20 of themselves (8 units of 2^-23), for tables of any first
entry: where one symbol has nearly all of the weight, the entropy is as small as what the others have, and nothing of the largest
may add to it."""

import numpy as np
import pytest

from taco_amd import synth
from tests import paged_ref as ref
from tests.test_gpu_tree_cache import Gpu

pytestmark = pytest.mark.gpu

FIRST = [5 ** 17, 41, 10 ** 12, 2 ** 40 - 1, 12_345_677, 3, 2 ** 40]


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


def check_entropies(gpu, logits, table):
    rows, vocab = logits.shape
    print(f"entropies {rows}x{vocab} {logits.dtype} of {len(table)} entries from {int(table[0])}", flush=True)
    out = np.full(rows, 7, np.float32)
    held = gpu(out)
    gpu.hip.score_tokens(gpu.dev, gpu(logits), None, gpu(table), (rows, vocab, len(table)), 0, None, None, held, None, None,
                         bits=8 * logits.dtype.itemsize)
    ref.close(gpu.back(held, out), ref.scores(logits, table, None, 0)[2], 8)


# vocabularies of each form: a wave, eight, registers of whole logits, of 16 bits each, longer
@pytest.mark.parametrize("dtype", [np.int32, np.int64])
@pytest.mark.parametrize("vocab", [2, 900, 9000, 50_257, 99_999, 150_000])
def test_one_symbol_with_nearly_all_the_weight(gpu, vocab, dtype):
    for first in FIRST:
        table = np.maximum(np.rint(float(first) * np.exp(-np.arange(4000) / 100)), 0).astype(np.uint64)
        table[0] = first
        logits = np.full((8, vocab), -9000, dtype)       # past the table's end, whose entry is small or 0
        for i, distance in enumerate((9000, 3999, 3500, 2700, 1400, 700, 100, 1)):
            logits[i, -1] = 0
            logits[i, 0] = -distance                     # one other symbol that counts
        check_entropies(gpu, logits, table)
        check_entropies(gpu, logits, np.array([first, first, 1], np.uint64))  # a second entry as large as the first
        check_entropies(gpu, logits, np.array([first, 1], np.uint64))


@pytest.mark.parametrize("first", [5 ** 17, 41, 2 ** 40])
def test_through_a_batch(first, monkeypatch):
    """Models whose tables fall from the first entry to 1 at once, so that most rows have one symbol that counts."""
    from taco_amd import hip
    both = synth.exp_tables
    monkeypatch.setattr(synth, "exp_tables", lambda n: (both(n)[0], np.concatenate([[first], np.ones(n - 1)]).astype(np.uint64)))
    model = hip.HipModel.load(hip.HipDevice.open(0), synth.build_model(synth.Dims(1, 2, 64, 128)))
    inputs = [(s, int(x)) for s in range(2) for x in np.random.default_rng(1).integers(0, model.vocab_size(), 9)]
    plain, scored = (hip.HipBatch(model, 2, 32) for _ in range(2))
    want = []
    for w in plain.run_weights(inputs):
        share = w.astype(np.float64) / w.sum()
        want.append((share * np.log1p((w.sum() - w).astype(np.float64) / w.astype(np.float64))).sum())
    ref.close(scored.run_scored(inputs).entropy, np.array(want), 8)


@pytest.mark.parametrize("weight", [348_605, 2 ** 20 - 1, 10 ** 6 + 3, 77_777])
@pytest.mark.parametrize("step,most", [(64, 254), (512, 31), (1024, 15)])
def test_equal_terms_in_one_lane(gpu, step, most, weight):
    """Many equal terms whose bins lie a workgroup's lanes apart: a sum in 32 bits would round them all the same way."""
    table = np.full(16_384, weight, np.uint64)
    table[0] = 2 ** 40
    for each, far in ((4, 0), (3, 0), (1, 0), (4, 8000), (4, 40_000)):
        logits = -np.concatenate([[0], np.repeat(step * np.arange(1, most + 1), each)])
        logits = np.concatenate([logits, np.full(far, -20_000)])  # longer rows, in the forms of more waves
        check_entropies(gpu, np.resize(logits, (2, len(logits))).astype(np.int32), table)
        check_entropies(gpu, np.resize(logits, (2, len(logits))).astype(np.int64), table)
