"""Trees of drafted tokens through the batch, against the oracle's sessions: every node's weights and intervals
are those of the context and the path to it, run token by token; committed paths continue the context, with more
trees, plain inputs, truncations and restarts after them; and the refusals leave every position."""

import numpy as np
import pytest

from oracle import oracle as O
from tests.attention_ref import random_parents

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from taco_amd import hip
    return hip.HipDevice.open(0)


def path_to(parents, node):
    out = []
    while node >= 0:
        out.insert(0, node)
        node = parents[node]
    return out


def rows_after(om, k, inputs, count):
    """The weights after each of the last `count` inputs of a stream that starts with EOT."""
    if len(inputs) <= om.n_ctx:  # no restart: the fast path's window (row i follows i + 1 inputs)
        return O.fast_window_weights(om, inputs[1:] + [0])[len(inputs) - count:]
    s = O.Session(om, k)
    rows = [s.start_block()] + [s.step(t) for t in inputs[1:]]
    return rows[len(inputs) - count:]


def want_rows(om, k, context, tokens, parents):
    """The weights of each node of a tree after the inputs `context`: a stream for each leaf."""
    rows = [None] * len(tokens)
    for leaf in set(range(len(tokens))) - set(parents):
        path = path_to(parents, leaf)
        for node, row in zip(path, rows_after(om, k, context + [tokens[i] for i in path], len(path))):
            rows[node] = row
    return rows


def check(dev, model_bytes, slots, n_ctx, vocab, k, rounds, nodes, seed, max_rows=None, prompt=None):
    from taco_amd import hip
    om, hm = O.Model(model_bytes), hip.HipModel.load(dev, model_bytes)
    r = np.random.default_rng(seed)
    batch = hip.HipBatch(hm, slots, max_rows or max(64, slots * nodes, prompt or 0))
    batch.set_overlap(k)
    streams = [[hm.eot_token()] + [int(x) for x in r.integers(0, vocab - 1, r.integers(0, prompt or n_ctx // 2))]
               for _ in range(slots)]
    batch.run_without_readback([(s, t) for s in range(slots) for t in streams[s]])
    for _ in range(rounds):
        inputs, parents, of = [], [], {}
        for s in range(slots):
            room = n_ctx - batch.position(s)
            count = min(int(r.integers(1, nodes + 1)), room)
            if count:
                of[s] = ([int(x) for x in r.integers(0, vocab - 1, count)], random_parents(r, count), [])
        # the slots' nodes interleaved, each slot's in order
        left = {s: 0 for s in of}
        while left:
            s = int(r.choice(list(left)))
            tokens, ps, at = of[s]
            i = left[s]
            inputs.append((s, tokens[i]))
            parents.append(at[ps[i]] if ps[i] >= 0 else -1)
            at.append(len(inputs) - 1)
            left[s] += 1
            if left[s] == len(tokens):
                del left[s]
        before = [batch.position(s) for s in range(slots)]
        got = batch.run_tree_weights(inputs, parents)
        assert [batch.position(s) for s in range(slots)] == before
        paths = {}
        for s, (tokens, ps, at) in of.items():
            want = want_rows(om, k, streams[s], tokens, ps)
            for i, row in enumerate(want):
                assert np.array_equal(got[at[i]], row), (s, i)
            if r.random() < 0.8:
                paths[s] = path_to(ps, int(r.integers(0, len(tokens)))) if r.random() < 0.9 else []
        if r.random() < 0.5:  # the same trees again, coded
            queries = [(0, int(x)) for x in r.integers(0, vocab, len(inputs))]
            raw = batch.run_tree_coded_raw(inputs, parents, queries, 32)
            for row, w, (_, token) in zip(raw, got, queries):
                assert (int(row[0]), int(row[1]), int(row[2])) == (token, *O.freq_interval(w, 32, token))
        batch.commit_paths(paths)
        for s, path in paths.items():
            streams[s] += [of[s][0][i] for i in path]
            assert batch.stream_len(s) == len(streams[s])
        s = int(r.integers(0, slots))
        if r.random() < 0.4 and len(streams[s]) > 3:  # back by a token or two
            streams[s] = streams[s][:-int(r.integers(1, 3))]
            batch.truncate(s, len(streams[s]))
        token = [(s, int(x)) for s, x in enumerate(r.integers(0, vocab - 1, slots))]
        got = batch.run_weights(token)
        for s, t in token:
            streams[s].append(t)
            assert np.array_equal(got[s], rows_after(om, k, streams[s], 1)[0]), s


def tiny(heads, d, n_ctx, layers=2, vocab=300):
    return (layers, heads, d, 2 * d, vocab, n_ctx)


@pytest.mark.parametrize("heads,d", [(4, 64), (2, 128), (3, 60), (1, 128), (2, 96)])  # head dims 16, 64, 20, 128, 48
def test_trees_equal_the_paths_run_alone(dev, heads, d):
    check(dev, O.build_model(tiny(heads, d, 64), 0x7EE0 + d, 64), 3, 64, 300, 0, 12, 9, seed=heads * d)


def test_trees_over_restarts(dev):
    """Streams of several contexts with overlap: trees up to a context's last place, then plain inputs that restart it,
    truncations back across a restart after a tree wrote over the old context's rows."""
    check(dev, O.build_model(tiny(2, 128, 40), 0x7EE1, 40), 4, 40, 300, 7, 30, 12, seed=5)


def test_trees_of_a_wide_model(dev):
    check(dev, O.build_model(O.tiny_dims(), 0x7AC0_0001, 64, wide=True), 2, 64, 300, 3, 10, 9, seed=6)


@pytest.mark.parametrize("n_ctx,prompt,nodes", [(256, 200, 40), (1024, 900, 70), (2400, 2200, 20)])
def test_trees_after_long_contexts(dev, n_ctx, prompt, nodes):
    from taco_amd import synth
    dims = synth.Dims(n_layer=1, n_head=2, d_model=128, d_ff=128, vocab=200, n_ctx=n_ctx)
    check(dev, synth.build_model(dims, seed=0x7EE2), 2, n_ctx, 200, 0, 2, nodes, seed=n_ctx, prompt=prompt, max_rows=2 * prompt)


def test_refusals_leave_every_position(dev):
    from taco_amd import hip
    hm = hip.HipModel.load(dev, O.build_model(tiny(2, 64, 64), 0x7EE3, 64))
    batch = hip.HipBatch(hm, 2, 100)
    batch.run_without_readback([(0, 1)] * 60 + [(1, 1)] * 3)

    def refused(error, fn, *args):
        with pytest.raises(error):
            fn(*args)
        assert [batch.position(0), batch.position(1)] == [60, 3]

    for parents in ([0], [1, -1], [-1, 2]):
        refused(hip.Unsupported, batch.run_tree_weights, [(1, 5)] * len(parents), parents)
    refused(hip.Unsupported, batch.run_tree_weights, [(1, 5), (0, 5)], [-1, 0])  # a parent of another slot
    refused(hip.Unsupported, batch.run_tree_weights, [(0, 5)] * 5, [-1] * 5)  # past the context
    refused(hip.Unsupported, batch.run_tree_weights, [(1, 5)] * 101, [-1] * 101)  # more than a pass
    refused(hip.LengthMismatch, batch.run_tree_weights, [(1, 5)], [])
    refused(hip.BadSlot, batch.run_tree_weights, [(2, 5)], [-1])
    refused(hip.ModelError, batch.run_tree_weights, [(1, 300)], [-1])
    refused(hip.Unsupported, batch.run_tree_coded_raw, [(1, 5)], [-1], [(0, 300)])
    refused(hip.Unsupported, batch.commit_paths, {1: [0]})  # no tree yet
    batch.run_tree_weights([(1, 5), (1, 6), (1, 7), (0, 4)], [-1, 0, 0, -1])
    for path in ([1], [0, 0], [0, 1, 2], [3], [0, 3]):
        refused(hip.Unsupported, batch.commit_paths, {1: path})
    refused(hip.Unsupported, batch.commit_paths, {0: [0], 1: [1]})  # one bad path: no slot moves
    refused(hip.BadSlot, batch.commit_paths, {2: []})
    batch.commit_paths({1: []})
    refused(hip.Unsupported, batch.commit_paths, {1: [0]})  # the tree is gone
    for drop in (lambda: batch.reset(0), lambda: batch.truncate(0, 60), lambda: batch.run_without_readback([(0, 1)])):
        batch.reset(0)
        batch.run_without_readback([(0, 1)] * 60)
        batch.run_tree_weights([(0, 4)], [-1])
        drop()
        with pytest.raises(hip.Unsupported):
            batch.commit_paths({0: [0]})
    assert batch.run_tree_weights([], []).shape == (0, 300)
    batch.commit_paths({})
