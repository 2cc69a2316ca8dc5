"""Paged caches with a scale for each page and head, and scores of tokens, as cases that a timing program can run.

A case is a dict of plain values. `kind` names the operator:

- append: hip.pages_append, keys and values of new tokens into the pages of a cache in 8 bits; the first row
          of a page sets its scale.
- attend: hip.attend_paged, attention of one token or of a causal chunk of tokens over such a cache.
- score:  hip.score_tokens, log probabilities and ranks of given tokens, the entropy and the top alternatives
          of rows of logits.

All but the logarithms are integers that the arithmetic fixes. With `own` false `run` computes it with elementary
torch operations, with `own` true by the framework's kernels.
"""

import numpy as np
import torch

own = False

_HEADROOM = 20  # sixteenths: the scale of a page holds values up to 1.25 times its first row's
_MAX_SCALE = 64
_SCORE_M, _OUT_M, _P = 33_000_000, 1_300_000_000, 24
_LEN = 8192  # entries of the attention's exponent table


def listed():
    return [
        # The decode step of 64 streams of the small model: one row each into its last page.
        {"name": "append-step", "kind": "append", "streams": 64, "t": 1, "kv_heads": 12, "head_dim": 64, "page": 64,
         "context": 1000, "bits": 16},
        # Chunks of prompts, ragged, into small pages.
        {"name": "append-chunks", "kind": "append", "streams": 16, "t": 255, "kv_heads": 16, "head_dim": 64,
         "page": 16, "context": 700, "bits": 16},
        # Whole windows of the small model.
        {"name": "append-windows", "kind": "append", "streams": 64, "t": 1024, "kv_heads": 12, "head_dim": 64,
         "page": 64, "context": 0, "bits": 16},
        # One token of one session.
        {"name": "attend-session", "kind": "attend", "streams": 1, "t": 1, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "page": 64, "context": 1000, "bits": 16},
        # The decode step of 64 streams of the small model.
        {"name": "attend-64x12", "kind": "attend", "streams": 64, "t": 1, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "page": 64, "context": 1024, "bits": 16},
        # GPT-2-XL heads over long caches, ragged.
        {"name": "attend-xl-long", "kind": "attend", "streams": 8, "t": 1, "heads": 25, "kv_heads": 25,
         "head_dim": 64, "page": 128, "context": 16384, "bits": 16},
        # Wide heads that share keys and values, small pages.
        {"name": "attend-shared", "kind": "attend", "streams": 32, "t": 1, "heads": 32, "kv_heads": 4,
         "head_dim": 128, "page": 16, "context": 4000, "bits": 16},
        # Chunks of prompts, ragged: each row sees the keys before it.
        {"name": "attend-chunks", "kind": "attend", "streams": 16, "t": 256, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "page": 64, "context": 1024, "bits": 16},
        # One token of a session: its score and drafts for the next ones.
        {"name": "score-session", "kind": "score", "rows": 1, "vocab": 50257, "bits": 64, "len": 8192, "top": 8},
        # The decode step of 64 streams.
        {"name": "score-64", "kind": "score", "rows": 64, "vocab": 50257, "bits": 32, "len": 8192, "top": 16},
        # A small vocabulary of an odd size, few steps in the table: many ties.
        {"name": "score-small", "kind": "score", "rows": 3001, "vocab": 299, "bits": 64, "len": 301, "top": 5},
        # Perplexity of whole windows.
        {"name": "score-windows", "kind": "score", "rows": 4096, "vocab": 50257, "bits": 32, "len": 8192, "top": 1},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "score", "score"])
    if kind == "score":
        vocab = _log_int(rng, 16, 131072)
        rows = _log_int(rng, 1, max(1, min(4096, 200_000_000 // vocab)))
        return {"kind": kind, "rows": rows, "vocab": vocab, "bits": rng.choice([32, 64]),
                "len": _log_int(rng, 64, 16384), "top": min(vocab, rng.choice([0, 1, 5, rng.randrange(1, 65)]))}
    kv_heads, hd = rng.choice([1, 4, 12, 16, 25]), rng.choice([64, 64, 64, 32, 128, 80])
    case = {"kind": kind, "kv_heads": kv_heads, "head_dim": hd, "page": rng.choice([16, 32, 64, 128]),
            "bits": rng.choice([16, 16, 8])}
    if kind == "append":
        t = rng.choice([1, _log_int(rng, 1, 1024)])
        streams = _log_int(rng, 1, max(1, min(256, 50_000_000 // (t * kv_heads * hd))))
        return {**case, "streams": streams, "t": t, "context": rng.choice([0, _log_int(rng, 1, 2000)])}
    group = rng.choice([1, 1, 1, 2, 4, 8])
    t = rng.choice([1, 1, _log_int(rng, 2, 256)])
    context = max(t, _log_int(rng, 16, 16384))
    most = min(210_000_000 // (context * kv_heads * hd), 50_000_000 // (context * kv_heads * t * group))
    streams = _log_int(rng, 1, max(1, min(64, most)))
    return {**case, "streams": streams, "t": t, "heads": kv_heads * group, "context": context}


# ---- inputs ------------------------------------------------------------------------------------


def _exp_table(length, bits, step=256.0):
    """round(2^bits exp(-i / step))"""
    return np.rint(2.0 ** bits * np.exp(-np.arange(length) / step))


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _ragged(r, lo, hi, n):
    """n lengths in lo ..= hi, the first the largest."""
    x = r.integers(lo, hi + 1, n).astype(np.int32)
    x[0] = hi
    return x


def _rows(case, g, shape):
    """Values of new tokens: heavy tails and a few large channels, as attention's keys have; 16 bits or 8."""
    x = torch.randn(shape, device="cuda", generator=g)
    x *= 1 + 4 * (torch.rand(shape[-2:], device="cuda", generator=g) < 0.05)
    if case["bits"] == 8:
        return (x * 30).round_().clamp_(-127, 127).to(torch.int8)
    return (x * 300).round_().clamp_(-32767, 32767).to(torch.int16)


def _pool(case, seed, keys):
    """A pool of pages (the last one is spare: no table names it) and the table of the streams' pages."""
    r = np.random.default_rng(seed)
    b, page = case["streams"], case["page"]
    width = -(-keys // page)
    pages = b * width + b // 8 + 1
    table = r.permutation(pages)[:b * width].reshape(b, width).astype(np.int32)
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (pages + 1, case["kv_heads"], page, case["head_dim"])
    k, v = (torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
    if case["bits"] == 8:
        ks, vs = (torch.ones(shape[:2], dtype=torch.int32, device="cuda") for _ in range(2))
    else:  # over a factor of a few
        ks, vs = (torch.randn(shape[:2], device="cuda", generator=g).mul_(0.5).exp_().mul_(10).ceil_()
                  .clamp_(1, _MAX_SCALE).to(torch.int32) for _ in range(2))
    return r, g, {"case": case, "k": k, "v": v, "ks": ks, "vs": vs, "table": _cuda(table), "pages": pages,
                  "width": width}


def prepare(case, seed):
    kind = case["kind"]
    if kind == "score":
        r = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        rows, vocab, n = case["rows"], case["vocab"], case["top"]
        logits = torch.randn((rows, vocab), device="cuda", generator=g).mul_(min(700.0, case["len"] / 8))
        logits = logits.add_(12345.0).round_().to(torch.int64 if case["bits"] == 64 else torch.int32)
        # half of the tokens are likely ones
        likely = logits[:, :max(1, vocab // 2)].argmax(dim=1).to(torch.int32)
        some = _cuda(r.integers(0, vocab, rows).astype(np.int32))
        tokens = torch.where(_cuda(r.random(rows) < 0.5), likely, some)
        empty = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
        return {"case": case, "logits": logits, "tokens": tokens,
                "table": _cuda(_exp_table(case["len"], 40).astype(np.int64)),
                "logprob": empty(rows), "rank": empty(rows, dtype=torch.int32), "entropy": empty(rows),
                "top": empty(rows, n, dtype=torch.int32), "top_logprob": empty(rows, n)}
    b, t, context, hd = case["streams"], case["t"], case["context"], case["head_dim"]
    if kind == "append":
        r, g, s = _pool(case, seed, context + t)
        # keys and values lie side by side, as a projection of both leaves them
        kv = _rows(case, g, (b, t, 2, case["kv_heads"], hd))
        ctx = _ragged(r, context // 2, context, b)
        s.update(new_k=kv[:, :, 0], new_v=kv[:, :, 1], ctx=_cuda(ctx), rows=_cuda(_ragged(r, (t + 1) // 2, t, b)),
                 ctx_out=torch.zeros(b, dtype=torch.int32, device="cuda"))
        return s
    r, g, s = _pool(case, seed, context)
    rows = _ragged(r, (t + 1) // 2, t, b)
    s.update(q=torch.randint(-127, 128, (b, t, case["heads"], hd), dtype=torch.int8, device="cuda", generator=g),
             ctx=_cuda(np.maximum(_ragged(r, max(1, context // 2), context, b), rows)), rows=_cuda(rows),
             exp=_cuda(_exp_table(_LEN, 30).astype(np.int32)),
             out=torch.zeros((b, t, case["heads"], hd), dtype=torch.int8, device="cuda"))
    return s


def _shifts(case):
    """The shifts of the score and of the output: scores of a few nats (256 steps each), outputs of about 20."""
    return (35, 56) if case["bits"] == 16 else (32, 53)


# ---- the framework's kernels ---------------------------------------------------------------------

_handle = None


def _device():
    global _handle
    if _handle is None:
        from taco_amd import hip
        _handle = (hip, hip.HipDevice.open(0))
    return _handle


def _run_own(s):
    hip, dev = _device()
    c = s["case"]
    if c["kind"] == "score":
        hip.score_tokens(dev, s["logits"], s["tokens"], s["table"], (c["rows"], c["vocab"], c["len"]), c["top"],
                         s["logprob"], s["rank"], s["entropy"], s["top"], s["top_logprob"])
        return _scores(s)
    cache = hip.PagedCache(s["k"], s["v"], s["ks"], s["vs"], s["pages"], c["kv_heads"], c["page"], c["head_dim"],
                           _MAX_SCALE)
    b, t, w = c["streams"], c["t"], s["width"]
    if c["kind"] == "append":
        hip.pages_append(dev, cache, s["new_k"], s["new_v"], s["table"], s["ctx"], s["rows"], (b, t, w), _HEADROOM,
                         s["ctx_out"])
        return _pages(s)
    score_s, out_s = _shifts(c)
    rule = hip.AttentionRule(_SCORE_M, score_s, _OUT_M, out_s, s["exp"], _LEN, _P)
    hip.attend_paged(dev, cache, s["q"], s["table"], s["ctx"], s["rows"], (b, t, c["heads"], w, c["context"]), rule,
                     s["out"])
    return s["out"]


def _scores(s):
    return {k: s[k] for k in ("logprob", "rank", "entropy", "top", "top_logprob")}


def _pages(s):
    """Without the spare page."""
    return {**{k: s[k][:s["pages"]] for k in ("k", "v", "ks", "vs")}, "ctx": s["ctx_out"]}


# ---- the plain forms -----------------------------------------------------------------------------


def _plain_append(s):
    c, ctx = s["case"], s["ctx"].long()[:, None]
    page, spare = c["page"], s["pages"]
    i = torch.arange(c["t"], device="cuda")[None]
    at = ctx + i  # [b, t]
    live = i < s["rows"].long()[:, None]
    number = torch.gather(s["table"].long(), 1, (at // page).clamp(max=s["width"] - 1))
    number = torch.where(live, number, spare)
    first = at // page * page - ctx  # the page's first row in this call, below 0: before it
    for x, pool, scales in ((s["new_k"], s["k"], s["ks"]), (s["new_v"], s["v"], s["vs"])):
        if c["bits"] == 8:
            scale = torch.ones(x.shape[:3], dtype=torch.int32, device="cuda")
            stored = x
        else:
            x = x.int()
            most = x.abs().amax(dim=-1)  # [b, t, h]
            fresh = ((most * _HEADROOM + 127 * 16 - 1) // (127 * 16)).clamp(1, _MAX_SCALE)
            fresh = torch.gather(fresh, 1, first.clamp(min=0)[..., None].expand(fresh.shape))
            scale = torch.where(first[..., None] >= 0, fresh, scales[number].clamp(1, _MAX_SCALE))
            wide = scale[..., None]
            stored = torch.div(2 * x + wide, 2 * wide, rounding_mode="floor").clamp(-127, 127).to(torch.int8)
        # rows that are no page's first write their scale to the spare page
        scales[torch.where(first == i, number, spare)] = scale
        pool[number, :, at % page] = stored
    torch.add(s["ctx"], s["rows"], out=s["ctx_out"])
    return _pages(s)


def _plain_attend(s):
    c, ctx, rows = s["case"], s["ctx"].long(), s["rows"].long()
    b, t, h, kvh, hd, keys = c["streams"], c["t"], c["heads"], c["kv_heads"], c["head_dim"], c["context"]
    group = h // kvh
    score_s, out_s = _shifts(c)

    def dense(x):  # [b, kvh, keys, ...]
        return x[s["table"].long()].transpose(1, 2).flatten(2, 3)[:, :, :keys]

    def scales(x):  # [b, kvh, keys, 1]
        x = x[s["table"].long()].clamp(1, _MAX_SCALE).transpose(1, 2)
        return x.repeat_interleave(c["page"], dim=2)[:, :, :keys, None].long()

    q = s["q"].view(b, t, kvh, group, hd).permute(0, 2, 4, 1, 3).reshape(b, kvh, hd, t * group).float().contiguous()
    dots = torch.matmul(dense(s["k"]).float(), q).to(torch.int64)  # below 2^24: exact
    score = (dots * (scales(s["ks"]) * _SCORE_M) + (1 << (score_s - 1))) >> score_s
    score = score.clamp_(-(1 << 40), 1 << 40)
    key = torch.arange(keys, device="cuda")[None, :, None]
    row = torch.arange(t, device="cuda")[None]
    live = row < rows[:, None]  # [b, t]
    sees = (key < (ctx[:, None] - rows[:, None] + 1 + row)[:, None]) & live[:, None]
    sees = sees.repeat_interleave(group, dim=2)[:, None]
    most = torch.where(sees, score, -(1 << 41)).amax(dim=2, keepdim=True)
    e = s["exp"].to(torch.int64)[(most - score).clamp_(0, _LEN - 1)]
    e = torch.where(sees, e, 0)
    total = e.sum(dim=2, keepdim=True)
    w = torch.div((e * scales(s["vs"])) << _P, total.clamp(min=1), rounding_mode="floor")
    # below 2^38: exact in 64-bit floats
    wv = torch.matmul(w.transpose(2, 3).double().contiguous(), dense(s["v"]).double()).to(torch.int64)
    low = ((wv & 0xFFFF) * _OUT_M + (1 << (out_s - 1))) >> 16  # the product needs more than 64 bits: in two parts
    out = (((wv >> 16) * _OUT_M + low) >> (out_s - 16)).clamp_(-127, 127).to(torch.int8)
    out = out.view(b, kvh, t, group, hd).transpose(1, 2).reshape(b, t, h, hd)
    s["out"].copy_(torch.where(live[:, :, None, None], out, s["out"]))
    return s["out"]


def _log_share(w, total):
    """ln(w / total), also where it is close to 0; minus infinity for no weight"""
    w = w.double()
    return -torch.log1p((total.double() - w) / w)


def _plain_score(s):
    c = s["case"]
    logits = s["logits"].long()
    d = (logits.amax(dim=1, keepdim=True) - logits).clamp_(max=c["len"] - 1)
    w = s["table"][d]
    total = w.sum(dim=1, keepdim=True)
    share = _log_share(w, total)
    entropy = -torch.where(w > 0, w.double() / total.double() * share, 0.0).sum(dim=1)
    token = s["tokens"].long()[:, None]
    order = d * c["vocab"] + torch.arange(c["vocab"], device="cuda")
    s["rank"].copy_((order < torch.gather(order, 1, token)).sum(dim=1))
    s["logprob"].copy_(torch.gather(share, 1, token)[:, 0])
    s["entropy"].copy_(entropy)
    if c["top"]:
        best = torch.topk(order, c["top"], dim=1, largest=False, sorted=True).values % c["vocab"]
        s["top"].copy_(best)
        s["top_logprob"].copy_(torch.gather(share, 1, best))
    return _scores(s)


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "score": _plain_score}[state["case"]["kind"]](state)


# ---- work and exact results ------------------------------------------------------------------------


def work(case):
    if case["kind"] == "score":
        rows, n = case["rows"], case["rows"] * case["vocab"]
        return {"bytes": n * case["bits"] // 8 + rows * (16 + 8 * case["top"]) + 8 * case["len"], "flops": 2 * n}
    b, t, kvh, hd = case["streams"], case["t"], case["kv_heads"], case["head_dim"]
    rows = b * t * (1 if t == 1 else 0.75)
    if case["kind"] == "append":
        values = 2 * rows * kvh * hd
        return {"bytes": values * (case["bits"] // 8 + 1) + 2 * rows * kvh / min(case["page"], t) * 4,
                "flops": values}
    keys = max(t * 0.75, 0.75 * case["context"])
    return {"bytes": b * kvh * 2 * keys * hd + 2 * rows * case["heads"] * hd,
            "flops": 4 * rows * case["heads"] * (keys - (rows / b - 1) / 2) * hd}


def _exact_append(s, case):
    page = case["page"]
    for i in range(case["streams"]):
        n = int(s["ctx"][i])
        for j in range(int(s["rows"][i])):
            number, place = s["table"][i, (n + j) // page], (n + j) % page
            for x, pool, scales in ((s["new_k"], s["k"], s["ks"]), (s["new_v"], s["v"], s["vs"])):
                x = x[i, j].astype(np.int64)  # [h, hd]
                if place == 0:
                    most = np.abs(x).max(axis=1)
                    scales[number] = 1 if case["bits"] == 8 else np.clip(-(-most * _HEADROOM // 2032), 1, _MAX_SCALE)
                scale = np.clip(scales[number], 1, _MAX_SCALE).astype(np.int64)[:, None]
                pool[number, :, place] = x if case["bits"] == 8 else \
                    np.clip(np.floor_divide(2 * x + scale, 2 * scale), -127, 127)
        s["ctx_out"][i] = n + int(s["rows"][i])
    return {**{k: s[k][:s["pages"]] for k in ("k", "v", "ks", "vs")}, "ctx": s["ctx_out"]}


def _exact_attend(s, case):
    kvh, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    group = case["heads"] // kvh
    score_s, out_s = _shifts(case)
    table, out = s["exp"].astype(np.int64), s["out"]
    for i in range(case["streams"]):
        n, live = int(s["ctx"][i]), int(s["rows"][i])
        numbers = s["table"][i, :-(-n // page)]
        sees = np.arange(n)[None] <= (n - live + np.arange(live))[:, None]
        for j in range(kvh):
            k, v = (s[x][numbers, j].reshape(-1, hd)[:n].astype(np.float64) for x in ("k", "v"))
            sk, sv = (np.repeat(np.clip(s[x][numbers, j], 1, _MAX_SCALE).astype(np.int64), page)[:n] for x in ("ks", "vs"))
            for m in range(j * group, (j + 1) * group):
                dots = (s["q"][i, :live, m].astype(np.float64) @ k.T).astype(np.int64)
                score = (dots * sk * _SCORE_M + (1 << (score_s - 1))) >> score_s
                top = np.where(sees, score, np.iinfo(np.int64).min).max(axis=1, keepdims=True)
                e = np.where(sees, table[np.minimum(np.where(sees, top - score, 0), _LEN - 1)], 0)
                w = ((e * sv) << _P) // e.sum(axis=1, keepdims=True)
                total = (w.astype(np.float64) @ v).astype(np.int64).astype(object)
                out[i, :live, m] = np.clip((total * _OUT_M + (1 << (out_s - 1))) >> out_s, -127, 127).astype(np.int8)
    return out


def _exact_score(s, case):
    table = s["table"]
    for i, row in enumerate(s["logits"].astype(np.int64)):
        w = table[np.minimum(row.max() - row, len(table) - 1)]
        total, some = int(w.sum()), w > 0
        share = np.full(len(w), -np.inf)
        share[some] = -np.log1p((total - w[some]).astype(np.float64) / w[some].astype(np.float64))
        s["entropy"][i] = -(w[some].astype(np.float64) / total * share[some]).sum()
        order = np.argsort(np.minimum(row.max() - row, len(table) - 1), kind="stable")
        token = int(s["tokens"][i])
        s["rank"][i], s["logprob"][i] = int(np.nonzero(order == token)[0][0]), share[token]
        s["top"][i], s["top_logprob"][i] = order[:case["top"]], share[order[:case["top"]]]
    return {k: s[k] for k in ("logprob", "rank", "entropy", "top", "top_logprob")}


def exact(case, seed):
    kind = case["kind"]
    if kind == "score":
        if case["rows"] * case["vocab"] > 20_000_000:
            return None
    elif kind == "append":
        if case["streams"] * case["t"] > 50_000:
            return None
    else:
        rows = case["streams"] * case["heads"] * case["t"]
        if rows * case["context"] > 60_000_000 or rows * case["head_dim"] > 2_000_000:
            return None
    s = {k: x.cpu().numpy() if torch.is_tensor(x) else x for k, x in prepare(case, seed).items()}
    for k in ("logprob", "entropy", "top_logprob"):
        if k in s:
            s[k] = s[k].astype(np.float64)
    return {"append": _exact_append, "attend": _exact_attend, "score": _exact_score}[kind](s, case)
