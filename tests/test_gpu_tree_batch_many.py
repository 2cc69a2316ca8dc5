"""More rows in a tree call than one grid of the row form holds: 70,000 slots with a token each, and 256 nodes in the
last one, at a head dim that the fast forms do not take."""

import numpy as np
import pytest

from oracle import oracle as O
from tests.attention_ref import random_parents
from tests.test_gpu_tree_batch import want_rows

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_grid():
    from taco_amd import hip
    slots, nodes, heads, vocab, n_ctx = 70_000, 256, 4, 300, 300
    assert slots * nodes * heads > 1 << 26
    data = O.build_model((1, heads, 16, 32, vocab, n_ctx), 0x7EE5, n_ctx)
    om, hm = O.Model(data), hip.HipModel.load(hip.HipDevice.open(0), data)
    batch = hip.HipBatch(hm, slots, slots + nodes)
    eot, last, r = hm.eot_token(), slots - 1, np.random.default_rng(7)
    context = [eot] + [int(x) for x in r.integers(0, vocab - 1, 30)]
    batch.run_without_readback([(last, t) for t in context])
    print("context run", flush=True)
    tokens, parents = [int(x) for x in r.integers(0, vocab - 1, nodes)], random_parents(r, nodes)
    single = np.column_stack([np.arange(last), np.full(last, eot)]).astype(np.uint32)
    inputs = np.concatenate([single, np.column_stack([np.full(nodes, last), tokens]).astype(np.uint32)])
    above = np.concatenate([np.full(last, -1), [p if p < 0 else last + p for p in parents]])
    symbols = np.arange(len(inputs)) % vocab
    raw = batch.run_tree_coded_raw(inputs, above, np.column_stack([np.zeros_like(symbols), symbols]), 32)
    print("tree run", flush=True)
    first = O.fast_window_weights(om, [0])[0]  # the weights after EOT alone, for every slot but the last
    want = np.array([(s, *O.freq_interval(first, 32, s)) for s in range(vocab)], np.uint64)
    assert np.array_equal(raw[:last], want[symbols[:last]])
    rows = want_rows(om, 0, context, tokens, parents)
    for i in range(nodes):
        s = int(symbols[last + i])
        assert (int(raw[last + i][0]), int(raw[last + i][1]), int(raw[last + i][2])) == (s, *O.freq_interval(rows[i], 32, s)), i
