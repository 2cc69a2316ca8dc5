"""The operators of speculative trees and of bounded caches, as cases that a timing program can run.

A case is a dict of plain values. `kind` names the operator:

- tree:   hip.attend_tree, attention of a tree of drafted tokens over each stream's cache.
- mass:   hip.attend_mass, attention of one token or of a causal chunk of tokens that adds the
          weight each key received to a 64-bit accumulator.
- evict:  hip.cache_evict, a cache cut to its budget in place: the keys of the largest accumulated
          weights and the most recent ones stay.
- commit: hip.cache_commit, the rows of the accepted path of a tree moved behind the context.

Every result is an integer that the arithmetic fixes. With `own` false `run` computes it with
elementary torch operations, with `own` true by the framework's kernels.
"""

import math

import numpy as np
import torch

own = False

# rescales that give scores of a few nats (256 steps each) and outputs of about 40
_SCORE_M, _SCORE_S = 1_400_000_000, 36
_OUT_M, _OUT_S = 1_300_000_000, 59
_P = 30
_LEN = 8192  # entries of the exponent table


def listed():
    return [
        # One session checks a small tree of drafts a little way into its context: latency.
        {"name": "tree-session", "kind": "tree", "streams": 1, "nodes": 8, "heads": 12, "head_dim": 64, "cap": 1024,
         "context": 100},
        # Decompression of 64 blocks of the small model, 16 drafts each, ragged contexts.
        {"name": "tree-64x16", "kind": "tree", "streams": 64, "nodes": 16, "heads": 12, "head_dim": 64, "cap": 1024,
         "context": 1000},
        # Wider heads, an odd number of drafts, contexts past 1,024.
        {"name": "tree-heads128", "kind": "tree", "streams": 16, "nodes": 23, "heads": 8, "head_dim": 128,
         "cap": 2048, "context": 2000},
        # GPT-2-XL heads, large trees over long caches.
        {"name": "tree-xl-long", "kind": "tree", "streams": 8, "nodes": 64, "heads": 25, "head_dim": 64, "cap": 8192,
         "context": 8100},
        # One token of one session whose cache is watched for eviction.
        {"name": "mass-session", "kind": "mass", "streams": 1, "rows": 1, "heads": 12, "head_dim": 64, "cap": 1024,
         "context": 1000, "ragged": False},
        # The decode step of 64 streams of the small model.
        {"name": "mass-64x12", "kind": "mass", "streams": 64, "rows": 1, "heads": 12, "head_dim": 64, "cap": 1024,
         "context": 1024, "ragged": False},
        # Chunks of prompts, ragged: each row sees the keys before it.
        {"name": "mass-prefill", "kind": "mass", "streams": 16, "rows": 256, "heads": 12, "head_dim": 64,
         "cap": 1024, "context": 1024, "ragged": True},
        # One session at its budget, one layer.
        {"name": "evict-session", "kind": "evict", "layers": 1, "streams": 1, "heads": 12, "head_dim": 64,
         "cap": 1024, "budget": 512, "recent": 128},
        # All layers of the small model, 64 streams, a quarter of the context given up.
        {"name": "evict-64", "kind": "evict", "layers": 12, "streams": 64, "heads": 12, "head_dim": 64, "cap": 1024,
         "budget": 768, "recent": 64},
        # Long caches cut to a quarter.
        {"name": "evict-long", "kind": "evict", "layers": 4, "streams": 4, "heads": 16, "head_dim": 64,
         "cap": 16384, "budget": 4096, "recent": 511},
        # One session accepts a path, all layers of the small model.
        {"name": "commit-session", "kind": "commit", "layers": 12, "streams": 1, "nodes": 8, "heads": 12,
         "head_dim": 64, "cap": 1024},
        # 64 streams of the medium model.
        {"name": "commit-64", "kind": "commit", "layers": 24, "streams": 64, "nodes": 32, "heads": 16,
         "head_dim": 64, "cap": 512},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "mass", "mass", "evict", "commit"])
    heads, hd = rng.choice([4, 12, 16, 25]), rng.choice([64, 64, 64, 32, 128, 80])
    if kind == "evict":
        cap = _log_int(rng, 64, 16384)
        layers = _log_int(rng, 1, 12)
        streams = _log_int(rng, 1, max(1, min(64, 9_000_000 // (layers * heads * cap) * 64 // hd)))
        budget = max(1, int(cap * rng.uniform(0.2, 0.95)))
        return {"kind": kind, "layers": layers, "streams": streams, "heads": heads, "head_dim": hd, "cap": cap,
                "budget": budget, "recent": int(budget * rng.choice([0, 0.1, 0.25, 0.5, 1]))}
    if kind == "commit":
        layers, streams, nodes = _log_int(rng, 1, 24), _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        cap = nodes + _log_int(rng, 16, 400)
        return {"kind": kind, "layers": layers, "streams": streams, "nodes": nodes, "heads": rng.choice([4, 12]),
                "head_dim": rng.choice([64, 64, 32, 80]), "cap": cap}
    rows = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 2, 64)]) if kind == "mass" else _log_int(rng, 1, 64)
    cap = rows + _log_int(rng, 16, 8000)
    most = 64 * 8192 * 200 * 64 // (rows * cap * heads * hd)
    streams = _log_int(rng, 1, max(1, min(64, most)))
    case = {"kind": kind, "streams": streams, "heads": heads, "head_dim": hd, "cap": cap}
    if kind == "tree":
        return {**case, "nodes": rows, "context": rng.choice([0, cap - rows, rng.randrange(1, cap - rows + 1)])}
    return {**case, "rows": rows, "context": rng.choice([cap, rng.randrange(rows, cap + 1)]),
            "ragged": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------------------------


def _table():
    return np.rint(2.0 ** 30 * np.exp(-np.arange(_LEN) / 256.0)).astype(np.int32)


def _caches(case, seed, layers):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (*layers, case["streams"], case["heads"], case["cap"], case["head_dim"])
    return [torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g) for _ in range(2)]


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _ragged(r, lo, hi, n):
    """n lengths in lo ..= hi, the first the largest."""
    x = r.integers(lo, hi + 1, n).astype(np.int32)
    x[0] = hi
    return x


def _trees(r, streams, t):
    """The node counts and the ancestor masks [streams, t, words] of random trees: most drafts hang on
    one of the last few nodes, some start at the context's end."""
    nodes = _ragged(r, (t + 1) // 2, t, streams)
    words = (t + 63) // 64
    sees = np.zeros((streams, t, 64 * words), bool)
    back = r.integers(1, 5, (streams, t))
    at = np.arange(streams)
    for i in range(t):
        parent = i - back[:, i]
        sees[:, i] = np.where((parent >= 0)[:, None], sees[at, np.maximum(parent, 0)], False)
        sees[:, i, i] = True
    mask = np.packbits(sees, axis=-1, bitorder="little").view(np.int64)
    return nodes, mask


def _attend_state(case, seed, rows):
    r = np.random.default_rng(seed)
    b, h, hd = case["streams"], case["heads"], case["head_dim"]
    k, v = _caches(case, seed, ())
    return r, {"case": case, "k": k, "v": v, "table": _cuda(_table()),
               "q": _cuda(r.integers(-127, 128, (b, rows, h, hd), dtype=np.int8)),
               "out": torch.zeros((b, rows, h, hd), dtype=torch.int8, device="cuda")}


def prepare(case, seed):
    kind, b, cap = case["kind"], case["streams"], case["cap"]
    if kind == "tree":
        r, s = _attend_state(case, seed, case["nodes"])
        nodes, mask = _trees(r, b, case["nodes"])
        ctx = _ragged(r, case["context"] // 2, case["context"], b)
        s.update(ctx=_cuda(ctx), nodes=_cuda(nodes), mask=_cuda(mask))
        return s
    if kind == "mass":
        t = case["rows"]
        r, s = _attend_state(case, seed, t)
        rows = _ragged(r, (t + 1) // 2, t, b) if case["ragged"] else np.full(b, t, np.int32)
        ctx = np.maximum(_ragged(r, max(1, case["context"] // 2), case["context"], b), rows)
        s.update(ctx=_cuda(ctx), rows=_cuda(rows),
                 mass=torch.zeros((b, case["heads"], cap), dtype=torch.int64, device="cuda"))
        return s
    r = np.random.default_rng(seed)
    k, v = _caches(case, seed, (case["layers"],))
    s = {"case": case, "k": k, "v": v, "ctx_out": torch.zeros(b, dtype=torch.int32, device="cuda")}
    if kind == "evict":
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        shape = k.shape[:-1]
        # weights over a few orders of magnitude, some keys without any
        mass = (torch.randn(shape, device="cuda", generator=g).mul_(2).exp_().mul_(2.0 ** 28)).to(torch.int64)
        mass[torch.rand(shape, device="cuda", generator=g) < 0.05] = 0
        s.update(mass=mass, mass_out=torch.zeros_like(mass), ctx=_cuda(_ragged(r, (cap + 1) // 2, cap, b)),
                 kept=torch.zeros((*shape[:-1], case["budget"]), dtype=torch.int32, device="cuda"))
        return s
    t = case["nodes"]
    accepted = _ragged(r, 0, max(1, t // 4), b)
    path = np.sort(np.argsort(r.random((b, t)), axis=1), axis=1)  # all nodes; then ascending choices of them
    pick = np.argsort(r.random((b, t)), axis=1)
    ones = np.arange(t)[None] < accepted[:, None]
    chosen = np.where(ones, pick, t)
    chosen.sort(axis=1)
    path = np.where(ones, chosen, path)
    s.update(path=_cuda(path.astype(np.int32)), accepted=_cuda(accepted), ctx=_cuda(_ragged(r, 0, cap - t, b)))
    return s


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
    b, h, hd, cap = c["streams"], c["heads"], c["head_dim"], c["cap"]
    if c["kind"] in ("tree", "mass"):
        rule = hip.AttentionRule(_SCORE_M, _SCORE_S, _OUT_M, _OUT_S, s["table"], _LEN, _P)
        if c["kind"] == "tree":
            hip.attend_tree(dev, s["q"], s["k"], s["v"], s["ctx"], s["nodes"], s["mask"], (b, c["nodes"], h, hd, cap),
                            rule, s["out"])
            return s["out"]
        hip.attend_mass(dev, s["q"], s["k"], s["v"], s["ctx"], s["rows"], s["mass"], (b, c["rows"], h, hd, cap), rule,
                        s["out"])
        return {"out": s["out"], "mass": s["mass"]}
    k, v = s["k"], s["v"]  # one tensor of all layers
    if c["kind"] == "evict":
        hip.cache_evict(dev, k, v, s["mass"], s["ctx"], (b, h, hd, cap), c["budget"], c["recent"], s["mass_out"],
                        s["ctx_out"], s["kept"])
    else:
        hip.cache_commit(dev, k, v, s["ctx"], s["path"], s["accepted"], (b, c["nodes"], h, hd, cap), s["ctx_out"])
    return _moved(s)


def _moved(s):
    out = {"k": s["k"], "v": s["v"], "ctx": s["ctx_out"]}
    if "kept" in s:
        out.update(mass=s["mass_out"], kept=s["kept"])
    return out


# ---- the plain forms -----------------------------------------------------------------------------


def _attend(s, sees):
    """The attention of rows [b, t, h, hd] with sees [b, 1, cap, t]: (p [b, h, cap, t], out [b, t, h, hd])."""
    q = s["q"].permute(0, 2, 3, 1).float().contiguous()  # [b, h, hd, t]
    dots = torch.matmul(s["k"].float(), q).to(torch.int64)  # below 2^24: exact
    score = ((dots * _SCORE_M + (1 << (_SCORE_S - 1))) >> _SCORE_S).clamp_(-(1 << 40), 1 << 40)
    most = torch.where(sees, score, -(1 << 41)).amax(dim=2, keepdim=True)
    e = s["table"].to(torch.int64)[(most - score).clamp_(0, _LEN - 1)]
    e = torch.where(sees, e, 0)
    total = e.sum(dim=2, keepdim=True)
    p = torch.div(e << _P, total.clamp(min=1), rounding_mode="floor")
    # below 2^38: exact in 64-bit floats
    pv = torch.matmul(p.transpose(2, 3).double().contiguous(), s["v"].double()).to(torch.int64)
    low = ((pv & 0xFFFF) * _OUT_M + (1 << (_OUT_S - 1))) >> 16  # the product needs more than 64 bits: in two parts
    out = (((pv >> 16) * _OUT_M + low) >> (_OUT_S - 16)).clamp_(-127, 127).to(torch.int8)
    return p, out.transpose(1, 2)


def _plain_tree(s):
    c, ctx = s["case"], s["ctx"].long()
    b, t, cap = c["streams"], c["nodes"], c["cap"]
    key = torch.arange(cap, device="cuda")[None, :, None]
    node = key - ctx[:, None, None]  # [b, cap, 1]
    at = node.clamp(0, t - 1)
    words = s["mask"].transpose(1, 2)  # [b, words, t]
    bits = torch.gather(words, 1, (at >> 6).expand(b, cap, t)) >> (at & 63)
    drafted = (node >= 0) & (node < s["nodes"][:, None, None]) & ((bits & 1) != 0)
    _, out = _attend(s, ((node < 0) | drafted)[:, None])
    live = torch.arange(t, device="cuda")[None] < s["nodes"][:, None]
    s["out"].copy_(torch.where(live[:, :, None, None], out, s["out"]))
    return s["out"]


def _plain_mass(s):
    c, ctx, rows = s["case"], s["ctx"].long(), s["rows"].long()
    key = torch.arange(c["cap"], device="cuda")[None, :, None]
    row = torch.arange(c["rows"], device="cuda")[None]
    live = row < rows[:, None]  # [b, t]
    sees = (key < (ctx[:, None] - rows[:, None] + 1 + row)[:, None]) & live[:, None]
    p, out = _attend(s, sees[:, None])
    s["mass"].add_(p.sum(dim=3))
    s["out"].copy_(torch.where(live[:, :, None, None], out, s["out"]))
    return {"out": s["out"], "mass": s["mass"]}


def _plain_evict(s):
    c, n = s["case"], s["ctx"].long()[:, None, None]  # [b, 1, 1]
    cap, budget, recent = c["cap"], c["budget"], c["recent"]
    heavy = budget - recent
    at = torch.arange(cap, device="cuda")
    full = n > budget
    masses = torch.where(at < n - recent, s["mass"], -1)
    order = torch.sort(masses, dim=-1, descending=True, stable=True).indices[..., :heavy]
    held = torch.zeros(s["mass"].shape, dtype=torch.bool, device="cuda").scatter_(-1, order, True)
    # the members at or above `heavy`, ascending, and the empty places' ranks
    movers = torch.sort(torch.where(held & (at >= heavy), at, cap), dim=-1).values
    empty = ~held & (at < heavy)
    mover = torch.gather(movers, -1, (torch.cumsum(empty, -1) - 1).clamp_(min=0)).clamp_(max=cap - 1)
    source = torch.where(at < heavy, torch.where(held, at, mover), n - recent + (at - heavy))
    source = torch.where(full, source, at)[..., :budget].clamp_(max=cap - 1)
    live = (at[:budget] < n).expand(source.shape)
    rows = source[..., None].expand(*source.shape, c["head_dim"])
    for x in (s["k"], s["v"]):
        x[..., :budget, :] = torch.where(live[..., None], torch.gather(x, -2, rows), x[..., :budget, :])
    moved = torch.where(live, torch.gather(s["mass"], -1, source), s["mass_out"][..., :budget])
    s["mass_out"].copy_(torch.where(at < n, 0, s["mass_out"]))
    s["mass_out"][..., :budget] = moved
    s["kept"].copy_(torch.where(live, source.to(torch.int32), s["kept"]))
    s["ctx_out"].copy_(s["ctx"].clamp(max=budget))
    return _moved(s)


def _plain_commit(s):
    c, ctx = s["case"], s["ctx"].long()[:, None]
    i = torch.arange(c["nodes"], device="cuda")[None]
    stream = torch.arange(c["streams"], device="cuda")[:, None]
    to = ctx + i
    source = torch.where(i < s["accepted"][:, None], ctx + s["path"], to)
    for x in (s["k"], s["v"]):
        x[:, stream, :, to] = x[:, stream, :, source]
    torch.add(s["ctx"], s["accepted"], out=s["ctx_out"])
    return _moved(s)


def run(state):
    if own:
        return _run_own(state)
    return {"tree": _plain_tree, "mass": _plain_mass, "evict": _plain_evict,
            "commit": _plain_commit}[state["case"]["kind"]](state)


# ---- work and exact results ------------------------------------------------------------------------


def work(case):
    kind, h, hd, b = case["kind"], case["heads"], case["head_dim"], case["streams"]
    if kind in ("tree", "mass"):
        context = 0.75 * case["context"]  # the mean of the contexts
        if kind == "tree":
            rows = 0.75 * case["nodes"]
            keys, seen = context + rows, context + 0.25 * rows
        else:
            rows = (0.75 if case["ragged"] else 1) * case["rows"]
            keys, seen = max(rows, context), max(rows, context) - (rows - 1) / 2
        # K and V once, the rows and the outputs; the accumulators read and written
        size = b * h * (2 * keys * hd + 2 * rows * hd + (16 * keys if kind == "mass" else 0))
        return {"bytes": size, "flops": 4 * b * h * rows * seen * hd}
    panels = case["layers"] * b * h
    if kind == "evict":
        n, budget, heavy = 0.75 * case["cap"], case["budget"], case["budget"] - case["recent"]
        share = min(1.0, max(0.0, (case["cap"] - budget) / (0.5 * case["cap"])))  # of streams above their budget
        n = 0.5 * (max(budget, case["cap"] / 2) + case["cap"]) if share < 1 else n
        others = max(1.0, n - case["recent"])
        moves = min(n - budget, case["recent"]) + heavy * max(0.0, others - heavy) / others
        return {"bytes": panels * (share * (moves * (4 * hd + 8) + 8 * (n - budget)) + 16 * n + 4 * budget),
                "flops": panels * n}
    moves = max(1, case["nodes"] // 4) / 2
    return {"bytes": panels * moves * 4 * hd + 4 * b * case["nodes"], "flops": panels * moves}


def _rescaled(x, m, s):
    return (x * m + (1 << (s - 1))) >> s


def _exact_rows(q, k, v, sees, table):
    """One head: q [t, hd], k, v [keys, hd], sees [t, keys]: the weights and the outputs."""
    dots = (q.astype(np.float64) @ k.astype(np.float64).T).astype(np.int64)
    score = np.clip(_rescaled(dots, _SCORE_M, _SCORE_S), -(1 << 40), 1 << 40)
    top = np.where(sees, score, np.iinfo(np.int64).min).max(axis=1, initial=np.iinfo(np.int64).min, keepdims=True)
    e = np.where(sees, table[np.minimum(np.where(sees, top - score, 0), _LEN - 1)], 0)
    p = (e << _P) // np.maximum(e.sum(axis=1, keepdims=True), 1)
    total = (p.astype(np.float64) @ v.astype(np.float64)).astype(np.int64).astype(object)
    return p, np.clip(_rescaled(total, _OUT_M, _OUT_S), -127, 127).astype(np.int8)


def exact(case, seed):
    kind, b, h, hd, cap = (case[k] for k in ("kind", "streams", "heads", "head_dim", "cap"))
    if kind in ("tree", "mass"):
        t = case["nodes" if kind == "tree" else "rows"]
        if b * h * t * cap > 30_000_000 or b * h * t * hd > 2_000_000:
            return None
        s = {k: x.cpu().numpy() for k, x in prepare(case, seed).items() if k != "case"}
        table, out = s["table"].astype(np.int64), s["out"]
        for i in range(b):
            n = int(s["ctx"][i])
            live = int(s["nodes" if kind == "tree" else "rows"][i])
            if kind == "tree":
                bits = np.unpackbits(s["mask"][i, :live].view(np.uint8), axis=1, bitorder="little")[:, :live]
                sees = np.concatenate([np.ones((live, n), bool), bits.astype(bool)], axis=1)
            else:
                sees = np.arange(n)[None] <= (n - live + np.arange(live))[:, None]
            keys = sees.shape[1]
            for j in range(h):
                p, out[i, :live, j] = _exact_rows(s["q"][i, :live, j], s["k"][i, j, :keys], s["v"][i, j, :keys], sees,
                                                  table)
                if kind == "mass":
                    s["mass"][i, j, :keys] += p.sum(axis=0)
        return out if kind == "tree" else {"out": out, "mass": s["mass"]}
    if case["layers"] * b * h * cap > 2_000_000:
        return None
    s = {k: x.cpu().numpy() for k, x in prepare(case, seed).items() if k != "case"}
    for i in range(b):
        n = int(s["ctx"][i])
        if kind == "commit":
            rows = n + s["path"][i, :s["accepted"][i]]
            for x in (s["k"], s["v"]):
                x[:, i, :, n:n + len(rows)] = x[:, i, :, rows].transpose(1, 2, 0, 3)
            s["ctx_out"][i] = n + len(rows)
            continue
        budget, heavy = case["budget"], case["budget"] - case["recent"]
        s["ctx_out"][i] = min(n, budget)
        for layer in range(case["layers"]):
            for j in range(h):
                at, mass = (layer, i, j), s["mass"][layer, i, j].copy()
                if n <= budget:
                    source = np.arange(n)
                else:
                    best = np.lexsort((np.arange(n - case["recent"]), -mass[:n - case["recent"]]))[:heavy]
                    source = np.arange(heavy)
                    source[np.setdiff1d(source, best)] = np.sort(best[best >= heavy])
                    source = np.concatenate([source, np.arange(n - case["recent"], n)])
                for x in (s["k"], s["v"]):
                    x[at][:len(source)] = x[at][source]
                s["mass_out"][at][:n] = 0
                s["mass_out"][at][:len(source)] = mass[source]
                s["kept"][at][:len(source)] = source
    return _moved(s)
