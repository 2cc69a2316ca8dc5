"""Plain 64-bit forms of the attention of several rows and of the cache operators, for the tests: numpy
integers, with Python's where a product passes 64 bits. Sums and products are exact, so every comparison
with a kernel is for equality."""

import numpy as np

LIMIT = 1 << 40


def rescale(x, m, s):
    """floor((x m + 2^(s - 1)) / 2^s) as Python integers; 0 past a shift of 95."""
    x = np.asarray(x).astype(object) * int(m)
    if s == 0:
        return x
    return x * 0 if s > 95 else (x + (1 << (s - 1))) >> s


def attend(q, k, v, sees, rule, table):
    """One head: q [t, hd], k, v [keys, hd] i8, sees [t, keys]. The weights p [t, keys] and out [t, hd] i8."""
    score_m, score_s, out_m, out_s, p_bits = rule
    t, keys = sees.shape
    if keys == 0:
        return np.zeros((t, 0), np.int64), np.zeros(q.shape, np.int8)
    dots = q.astype(np.int64) @ k.astype(np.int64).T
    product = dots * int(score_m)  # below 2^53
    s = int(score_s)
    score = product if s == 0 else (product * 0 if s > 62 else (product + (1 << (s - 1))) >> s)
    score = np.clip(score, -LIMIT, LIMIT)
    low = np.int64(-(1 << 62))
    top = np.where(sees, score, low).max(axis=1, keepdims=True)
    table = table.astype(np.int64)
    e = np.where(sees, table[np.minimum(np.where(sees, top - score, 0), len(table) - 1)], 0)
    total = e.sum(axis=1, keepdims=True)
    p = np.where(total > 0, (e << p_bits) // np.maximum(total, 1), 0)
    sums = p @ v.astype(np.int64)
    return p, np.clip(rescale(sums, out_m, out_s), -127, 127).astype(np.int8)


def tree(q, kc, vc, ctx, nodes, mask, rule, table, out):
    """hs_op_attend_tree_dev: q, out [b, t, h, hd], mask [b, t, words] u64; writes the live rows of out."""
    b, t, h, _ = q.shape
    cap = kc.shape[2]
    for s in range(b):
        n, live = min(int(ctx[s]), cap), min(int(nodes[s]) if nodes is not None else t, t)
        bits = np.unpackbits(np.ascontiguousarray(mask[s]).view(np.uint8), axis=1, bitorder="little")[:live, :live]
        sees = np.concatenate([np.ones((live, n), bool), bits.astype(bool)], axis=1)[:, :cap]
        for j in range(h):
            _, out[s, :live, j] = attend(q[s, :live, j], kc[s, j, :sees.shape[1]], vc[s, j, :sees.shape[1]], sees,
                                         rule, table)
    return out


def mass(q, kc, vc, ctx, rows, acc, rule, table, out):
    """hs_op_attend_mass_dev: adds to acc [b, h, cap] u64 and writes the live rows of out."""
    b, t, h, _ = q.shape
    cap = kc.shape[2]
    for s in range(b):
        n, live = min(int(ctx[s]), cap), min(int(rows[s]) if rows is not None else t, t)
        sees = np.arange(n)[None] <= (n - live + np.arange(live))[:, None]
        for j in range(h):
            p, out[s, :live, j] = attend(q[s, :live, j], kc[s, j, :n], vc[s, j, :n], sees, rule, table)
            acc[s, j, :n] += p.sum(axis=0).astype(np.uint64)
    return out


def evict(ks, vs, acc, ctx, budget, recent, acc_out, ctx_out, kept):
    """hs_op_cache_evict_dev on lists of caches [b, h, cap, hd]; acc, acc_out [layers, b, h, cap]."""
    cap, heavy = ks[0].shape[2], budget - recent
    for s in range(len(ctx)):
        n = min(int(ctx[s]), cap)
        ctx_out[s] = min(n, budget)
        for l, (k, v) in enumerate(zip(ks, vs)):
            for j in range(k.shape[1]):
                a = acc[l, s, j].copy()
                if n <= budget:
                    src = list(range(n))
                else:
                    order = sorted(range(n - recent), key=lambda i: (-int(a[i]), i))[:heavy]
                    stay = set(order)
                    movers = iter(sorted(i for i in order if i >= heavy))
                    src = [i if i in stay else next(movers) for i in range(heavy)] + list(range(n - recent, n))
                k[s, j, :len(src)] = k[s, j, src]
                v[s, j, :len(src)] = v[s, j, src]
                acc_out[l, s, j, :n] = 0
                acc_out[l, s, j, :len(src)] = a[src]
                if kept is not None:
                    kept[l, s, j, :len(src)] = src


def commit(ks, vs, ctx, path, accepted, ctx_out):
    """hs_op_cache_commit_dev on lists of caches [b, h, cap, hd]."""
    cap = ks[0].shape[2]
    for s in range(len(ctx)):
        n = int(ctx[s])
        rows = [n + int(x) for x in path[s, :int(accepted[s])]]
        ctx_out[s] = n + len(rows)
        to = [n + i for i, r in enumerate(rows) if r < cap and n + i < cap]
        rows = [r for i, r in enumerate(rows) if r < cap and n + i < cap]
        for x in ks + vs:
            x[s, :, to] = x[s, :, rows]


def random_parents(r, t, back=4):
    """Parents of a random tree of t nodes: -1 or one of the last `back` nodes before."""
    return [int(max(-1, i - r.integers(1, back + 1))) for i in range(t)]
