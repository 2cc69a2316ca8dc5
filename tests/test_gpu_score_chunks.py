"""Scores of more rows than the LM head takes at a time: those of the same inputs in calls of fewer rows, bit for bit."""

import numpy as np
import pytest

from taco_amd import synth

pytestmark = pytest.mark.gpu


def test_rows_of_several_chunks():
    from taco_amd import hip
    model = hip.HipModel.load(hip.HipDevice.open(0), synth.build_model(synth.Dims(1, 2, 64, 128)))
    r, slots = np.random.default_rng(5), 24
    V, n = model.vocab_size(), model.n_ctx() - 1
    assert V > 50_000 and slots * n > 2 * 1024
    at_once, apart = hip.HipBatch(model, slots, 4096), hip.HipBatch(model, slots, 256)
    inputs = [(s, int(x)) for s in range(slots) for x in r.integers(0, V, n)]
    tokens = r.integers(0, V, len(inputs))
    tokens[::7] = -1
    got = at_once.run_scored(inputs, tokens, 5)
    parts = [apart.run_scored(inputs[i:i + n], tokens[i:i + n], 5) for i in range(0, len(inputs), n)]
    for name in got._fields:
        assert np.array_equal(getattr(got, name), np.concatenate([getattr(p, name) for p in parts])), name
    assert [at_once.position(s) for s in range(slots)] == [n] * slots
