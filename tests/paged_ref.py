"""Plain 64-bit forms of the paged caches' operators and of the scores, for the tests: numpy integers, with Python's
where a product passes 64 bits, and 64-bit floats for the logarithms."""

import numpy as np

from tests.attention_ref import LIMIT, rescale


class Pool:
    """A pool of pages on the host, filled at random: what no call may touch, it has to keep."""

    def __init__(self, r, pages, kv_heads, page, hd, max_scale):
        self.shape, self.max_scale = (pages, kv_heads, page, hd), max_scale
        self.k, self.v = (r.integers(-127, 128, self.shape).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (r.integers(1, max_scale + 1, (pages, kv_heads)).astype(np.uint32) for _ in range(2))

    def arrays(self):
        return self.k, self.v, self.ks, self.vs


def append(pool, k, v, table, ctx, rows, headroom, ctx_out=None):
    """hs_op_pages_append_dev: k, v [b, t, kv_heads, hd] of int8 or int16."""
    pages, _, page, _ = pool.shape
    b, t = k.shape[:2]
    for s in range(b):
        n = min(int(ctx[s]), table.shape[1] * page)
        count = min(int(rows[s]) if rows is not None else t, t, table.shape[1] * page - n)
        for i in range(count):
            number, place = int(table[s, (n + i) // page]), (n + i) % page
            if number >= pages:
                continue
            for x, to, scales in ((k, pool.k, pool.ks), (v, pool.v, pool.vs)):
                row = x[s, i].astype(np.int64)
                if place == 0:
                    most = np.abs(row).max(axis=1)
                    scales[number] = 1 if x.dtype == np.int8 else np.clip(-(-most * headroom // 2032), 1, pool.max_scale)
                scale = np.clip(scales[number], 1, pool.max_scale).astype(np.int64)[:, None]
                to[number, :, place] = row if x.dtype == np.int8 else \
                    np.clip(np.floor_divide(2 * row + scale, 2 * scale), -127, 127)
        if ctx_out is not None:
            ctx_out[s] = n + count


def attend(pool, q, table, ctx, rows, keys, rule, exp, out):
    """hs_op_attend_paged_dev: q, out [b, t, heads, hd]; writes the live rows of out."""
    score_m, score_s, out_m, out_s, p_bits = rule
    pages, kv_heads, page, _ = pool.shape
    b, t, heads, hd = q.shape
    exp = exp.astype(np.int64)
    for s in range(b):
        n = min(int(ctx[s]), keys)
        live = min(int(rows[s]) if rows is not None else t, t)
        numbers = table[s, :-(-n // page)].astype(np.int64)
        held = np.minimum(numbers, pages - 1)
        sees = np.arange(n)[None] <= (n - live + np.arange(live))[:, None]
        sees = sees & np.repeat(numbers < pages, page)[None, :n]
        for h in range(heads):
            j = h // (heads // kv_heads)
            k, v = (x[held, j].reshape(-1, hd)[:n].astype(np.int64) for x in (pool.k, pool.v))
            ks, vs = (np.repeat(np.clip(x[held, j], 1, pool.max_scale).astype(np.int64), page)[:n] for x in (pool.ks, pool.vs))
            if n == 0:
                out[s, :live, h] = 0
                continue
            product = (q[s, :live, h].astype(np.int64) @ k.T) * (ks * int(score_m))  # below 2^53
            score = product if score_s == 0 else (product * 0 if score_s > 62 else (product + (1 << (score_s - 1))) >> score_s)
            score = np.clip(score, -LIMIT, LIMIT)
            top = np.where(sees, score, -(1 << 62)).max(axis=1, keepdims=True)
            e = np.where(sees, exp[np.minimum(np.where(sees, top - score, 0), len(exp) - 1)], 0)
            total = e.sum(axis=1, keepdims=True)
            w = np.where(total > 0, ((e * vs) << p_bits) // np.maximum(total, 1), 0)
            out[s, :live, h] = np.clip(rescale(w @ v, out_m, out_s), -127, 127).astype(np.int8)
    return out


def scores(logits, table, tokens, top):
    """hs_op_score_dev for rows of Python-sized integers: logprob, rank, entropy, top_tokens, top_logprob."""
    rows, vocab = logits.shape
    lp, rank, entropy = np.zeros(rows), np.full(rows, 0xFFFFFFFF, np.uint32), np.zeros(rows)
    tops, tops_lp = np.zeros((rows, top), np.uint32), np.zeros((rows, top))
    table = np.asarray(table).astype(np.uint64)
    for i in range(rows):
        # (differences as unsigned numbers: exact for any two logits)
        d = np.minimum(logits[i].max().astype(np.int64).view(np.uint64) - logits[i].astype(np.int64).view(np.uint64),
                       np.uint64(len(table) - 1)).astype(np.int64)
        lp[i], rank[i], entropy[i], tops[i], tops_lp[i] = scores_of(table[d], d, None if tokens is None else int(tokens[i]), top)
    return lp, rank, entropy, tops, tops_lp


def scores_of(w, d, token, top):
    """One row from its weights and the distances that order it."""
    total, some = int(w.sum()), w > 0
    share = np.full(len(w), -np.inf)
    share[some] = -np.log1p((np.uint64(total) - w[some]).astype(np.float64) / w[some].astype(np.float64))
    entropy = -(w[some].astype(np.float64) / total * share[some]).sum() if total else 0.0
    order = np.argsort(d, kind="stable")
    lp, rank = 0.0, 0xFFFFFFFF
    if token is not None and token < len(w):
        lp, rank = share[token], int(np.nonzero(order == token)[0][0])
    return lp, rank, entropy, order[:top], share[order[:top]]


def close(got, want, ulps):
    """float32 values within `ulps` units in the last place of the 64-bit ones (a unit is at most 2^-23 of the value),
    and equal infinities and zeros."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    finite = np.isfinite(want)
    assert np.array_equal(got[~finite], want[~finite])
    assert (np.abs(got[finite] - want[finite]) <= ulps * 2.0 ** -23 * np.abs(want[finite])).all(), \
        np.max(np.abs(got[finite] - want[finite]) / np.maximum(np.abs(want[finite]), 1e-300)) * 2.0 ** 23
