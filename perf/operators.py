"""Performance cases of the key-value cache and its attention: what is timed,
on which inputs, and what the results are.

The operators are rotary positions (alone, or fused with the write into the
cache's pages), attention of one new token over the paged cache, attention of
a prompt through a sliding window with a few first tokens that stay visible,
and the cache's page keeping (forking sequences, compacting the pool).

``listed`` names the cases, ``draw`` makes others of the same ranges,
``prepare`` makes what a program holds before the call and ``run`` makes the
call: with ``own`` through the package's public classes, without it as
elementary torch operations in 32 bits, rounded once at the end.  ``work``
states the bytes and operations a call cannot do without and ``exact``
evaluates the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEVICE = "cuda:0"

_opened = None


def _context():
    """The process's one device context, as an application opens it once."""
    global _opened
    if _opened is None:
        from vectorstorekit_amd import Context

        _opened = Context(0)
    return _opened


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # a decoding step of a few requests: the new tokens' queries and keys
        # get their positions; one launch's latency is what counts
        {"name": "rotary_step", "op": "rotary", "tokens": 8, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotated": 128, "layout": "half", "scaling": "none", "type": "bf16",
         "positions": 8192, "inverse": False},
        # a long prompt of a model stretched to a longer context
        {"name": "rotary_prompt", "op": "rotary", "tokens": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotated": 128, "layout": "half", "scaling": "yarn", "type": "bf16",
         "positions": 65536, "inverse": False},
        # ragged prompts rotated over half the head and written to the cache
        {"name": "append_prompts", "op": "append", "n": 24, "longest": 641, "page": 16,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotated": 64, "layout": "interleaved",
         "scaling": "linear", "type": "f16"},
        # one conversation's next token: latency
        {"name": "token_single", "op": "token", "n": 1, "longest": 777, "page": 16, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "bf16", "window": 0, "sinks": 0},
        # a serving batch of ragged contexts
        {"name": "token_batch", "op": "token", "n": 64, "longest": 8192, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "window": 0, "sinks": 0},
        # few very long contexts (retrieved documents): the length is split
        {"name": "token_long", "op": "token", "n": 3, "longest": 200003, "page": 128,
         "heads": 64, "kv_heads": 8, "dim": 128, "type": "f16", "window": 0, "sinks": 0},
        # every head with keys of its own, 32 bits, a window behind the sinks
        {"name": "token_window", "op": "token", "n": 17, "longest": 12001, "page": 32,
         "heads": 16, "kv_heads": 16, "dim": 96, "type": "f32", "window": 2048, "sinks": 4},
        # one short text through a small encoder-sized layer: latency
        {"name": "window_short", "op": "window", "n": 1, "longest": 333, "page": 0, "heads": 8,
         "kv_heads": 8, "dim": 64, "type": "f16", "window": 128, "sinks": 4},
        # a batch of ragged prompts, keys and values as the projections left them
        {"name": "window_ragged", "op": "window", "n": 8, "longest": 4096, "page": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "window": 1024, "sinks": 4},
        # one long prompt against the cache it was appended to
        {"name": "window_long", "op": "window", "n": 1, "longest": 16384, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "window": 4096, "sinks": 16},
        # a sampling step: branches dropped and forked anew from their parents
        {"name": "fork_branches", "op": "fork", "n": 48, "slots": 96, "longest": 2000,
         "pages": 8192, "page": 16, "layers": 4, "kv_heads": 8, "dim": 128, "type": "bf16"},
        # a half-empty pool packed before it is shrunk
        {"name": "compact_pool", "op": "compact", "slots": 64, "pages": 16384, "live": 8192,
         "moves": 4096, "page": 16, "layers": 2, "kv_heads": 8, "dim": 128, "type": "bf16"},
    ]


#: heads, heads of keys and values, and their dimension
HEADS = [(32, 8, 128), (16, 16, 64), (8, 1, 256), (12, 12, 96), (28, 4, 128), (20, 5, 80),
         (64, 8, 128), (9, 3, 64)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "token", "token", "token", "window", "window", "window",
                     "fork", "compact"])
    heads, kv_heads, dim = rng.choice(HEADS)
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    base = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "type": kind}
    page = rng.choice([16, 32, 64, 128])
    turn = {"rotated": rng.choice([dim, dim, dim // 2]), "layout": rng.choice(["half", "interleaved"]),
            "scaling": rng.choice(["none", "linear", "ntk", "yarn"])}
    if op == "rotary":
        most = int(16384 * 40 * 128 * 2 / ((heads + kv_heads) * dim * TYPES[kind].itemsize))
        return {**base, **turn, "tokens": _log(rng, 1, most), "inverse": rng.random() < 0.3,
                "positions": _log(rng, 4096, 131072)}
    if op == "append":
        n = _log(rng, 1, 64)
        return {**base, **turn, "n": n, "longest": _log(rng, 1, 16384 // n), "page": page}
    if op == "token":
        n = _log(rng, 1, 128)
        most = int(800e6 / (n * kv_heads * dim * TYPES[kind].itemsize))
        longest = _log(rng, 1, min(200000, most))
        window = rng.choice([0, 0, 0, _log(rng, 1, longest)])
        return {**base, "n": n, "longest": longest, "page": page, "window": window,
                "sinks": rng.choice([0, 1, 4, 16]) if window else 0}
    if op == "window":
        n = _log(rng, 1, 16)
        longest = _log(rng, 1, int(math.sqrt(16384 * 16384 * 32 * 128 / (n * heads * dim)) / 2))
        return {**base, "n": n, "longest": longest, "page": rng.choice([0, 0, page]),
                "window": _log(rng, 1, 4096), "sinks": rng.choice([0, 1, 4, 16])}
    per = page * kv_heads * dim * TYPES[kind].itemsize
    layers = rng.choice([1, 2, 4])
    del base["heads"]
    if op == "fork":
        slots, longest = _log(rng, 2, 128), _log(rng, 1, 2000)
        pages = 2 * slots * (longest // page + 1)
        while pages * per * layers > (1 << 30):
            slots, pages = slots // 2 + 1, pages // 2
            longest = max(1, pages // (2 * slots) * page - page)
        n = rng.randint(1, slots // 2)
        return {**base, "n": n, "slots": slots, "longest": longest,
                "pages": 2 * slots * (longest // page + 1), "page": page, "layers": layers}
    pages = _log(rng, 64, max(64, min(16384, (1 << 30) // (per * layers))))
    live = max(1, int(pages * rng.uniform(0.2, 0.8)))
    return {**base, "slots": rng.randint(1, 64), "pages": pages, "live": live,
            "moves": rng.randint(0, min(live, pages - live)), "page": page, "layers": layers}


# ------------------------------------------------------- what the cases stand on

def _lengths(case):
    """The sequences' lengths: ragged, the first the longest.  A case's own,
    whatever the seed, so that its work is known."""
    rng = random.Random(case["longest"] * 7919 + case["n"])
    top = case["longest"]
    return [top] + [1 + int((top - 1) * rng.random() ** 1.5) for _ in range(case["n"] - 1)]


def _frequencies(case):
    """Radians a position for each rotated pair, and the factor on the
    rotated part (64 bits)."""
    r, base, f = case["rotated"], 10000.0, 8.0
    i = np.arange(r // 2, dtype=np.float64)
    inv = base ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        return inv / f, 1.0
    if case["scaling"] == "ntk":
        return (base * f ** (r / (r - 2.0))) ** (-2.0 * i / r), 1.0
    if case["scaling"] == "yarn":
        def at(turns):
            return r * math.log(8192 / (2 * math.pi * turns)) / (2 * math.log(base))
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), r - 1)
        ramp = np.clip((i - low) / max(high - low, 1e-3), 0.0, 1.0)
        return inv * (1 - ramp) + inv / f * ramp, 0.1 * math.log(f) + 1.0
    return inv, 1.0


def _rotary(case):
    """The package's object for the same frequencies."""
    from vectorstorekit_amd import RotaryEmbedding

    scaling = {"none": None, "linear": {"type": "linear", "factor": 8.0},
               "ntk": {"type": "ntk", "factor": 8.0},
               "yarn": {"type": "yarn", "factor": 8.0, "original_length": 8192}}
    return RotaryEmbedding(_context(), case["dim"], rotary_dim=case["rotated"], base=10000.0,
                           layout=case["layout"], scaling=scaling[case["scaling"]])


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _projected(g, *shape, dtype):
    """Queries or keys as projections make them: some channels stand out."""
    x = torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)
    loud = 1.0 + 2.0 * (torch.rand(shape[-1], generator=g, device=DEVICE) < 0.05)
    return x.mul_(loud).to(dtype)


def _pool(g, case, layers=None):
    shape = (case["pages"], case["page"], case["kv_heads"], case["dim"])
    shape = shape if layers is None else (layers, *shape)
    t = TYPES[case["type"]]
    pool = [torch.empty(shape, device=DEVICE, dtype=t) for _ in range(2)]
    pool[0].copy_(_projected(g, *shape, dtype=t))
    pool[1].copy_(_normal(g, *shape, dtype=t))
    return pool


def _tables(g, lengths, page, pages, width):
    """A page table whose sequences hold pages from all over the pool."""
    used = [-(-x // page) for x in lengths]
    ids = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = np.full((len(lengths), width), -1, np.int64)
    at = 0
    for s, u in enumerate(used):
        table[s, :u] = np.arange(at, at + u)
        at += u
    where = torch.from_numpy(table).to(DEVICE)
    return torch.where(where >= 0, ids[where.clamp(min=0)], -1).to(torch.int32)


def _starts(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=DEVICE)


def _cache(case, s, refs=None):
    """The package's handle on a program's pages and tables."""
    from vectorstorekit_amd import PagedKVCache

    return PagedKVCache.over(_context(), s["k"], s["v"], s["table"], s["lengths"], refs)


def prepare(case, seed):
    g, op, t = _generator(seed), case["op"], TYPES[case["type"]]
    s = {"case": case, "op": op}
    if op in ("rotary", "append"):
        inv, amplitude = _frequencies(case)
        lengths = _lengths(case) if op == "append" else None
        tokens = case["tokens"] if op == "rotary" else sum(lengths)
        s["q"] = _projected(g, tokens, case["heads"], case["dim"], dtype=t)
        s["new_k"] = _projected(g, tokens, case["kv_heads"], case["dim"], dtype=t)
        # the table of cosines and sines that a program keeps
        span = case["positions"] if op == "rotary" else 2 * case["longest"]
        angle = torch.arange(span, dtype=torch.float64, device=DEVICE)[:, None] \
            * torch.from_numpy(inv).to(DEVICE)
        s["cos"], s["sin"] = ((f(angle) * amplitude).float() for f in (torch.cos, torch.sin))
        if op == "rotary":
            first = torch.randint(0, span, (1,), generator=g, device=DEVICE)
            s["positions"] = ((first + torch.arange(tokens, device=DEVICE)) % span
                              if tokens > 64 else
                              torch.randint(0, span, (tokens,), generator=g, device=DEVICE))
            s["positions"] = s["positions"].to(torch.int32)
        else:
            # each sequence has as much again in the cache already
            s["new_v"] = _normal(g, tokens, case["kv_heads"], case["dim"], dtype=t)
            s["starts"], s["longest"] = _starts(lengths), case["longest"]
            held = [2 * x for x in lengths]
            width = -(-max(held) // case["page"])
            pages = sum(-(-x // case["page"]) for x in held) + 3
            s["k"], s["v"] = _pool(g, {**case, "pages": pages})
            s["table"] = _tables(g, held, case["page"], pages, width)
            s["lengths"] = torch.tensor(held, dtype=torch.int32, device=DEVICE)
        if own:
            s["rotary"] = _rotary(case)
    elif op in ("token", "window"):
        lengths = _lengths(case)
        s["longest"], s["scale"] = case["longest"], case["dim"] ** -0.5
        tokens = case["n"] if op == "token" else sum(lengths)
        s["q"] = _projected(g, tokens, case["heads"], case["dim"], dtype=t)
        s["starts"] = _starts(lengths if op == "window" else [1] * case["n"])
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        if case["page"]:
            width = -(-max(lengths) // case["page"])
            pages = sum(-(-x // case["page"]) for x in lengths) + 3
            s["k"], s["v"] = _pool(g, {**case, "pages": pages})
            s["table"] = _tables(g, lengths, case["page"], pages, width)
        else:
            s["k"] = _projected(g, tokens, case["kv_heads"], case["dim"], dtype=t)
            s["v"] = _normal(g, tokens, case["kv_heads"], case["dim"], dtype=t)
    elif op == "fork":
        rng = random.Random(seed)
        s["k"], s["v"] = _pool(g, case, case["layers"])
        slots, n, page = case["slots"], case["n"], case["page"]
        kept = slots - n
        lengths = (_lengths({"n": kept, "longest": case["longest"]}) + [0] * n)
        width = -(-(case["longest"] + page) // page)
        s["table"] = _tables(g, lengths, page, case["pages"], width)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        s["refs"] = torch.zeros(case["pages"], dtype=torch.int32, device=DEVICE)
        held = s["table"][s["table"] >= 0].long()
        s["refs"][held] = 1
        # the slots dropped are the last ones, in an order of their own
        order = list(range(kept, slots))
        rng.shuffle(order)
        s["children"] = torch.tensor(order, dtype=torch.int32, device=DEVICE)
        parents = [rng.randrange(kept) if i else 0 for i in range(n)]
        s["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEVICE)
        _fork(s)  # the branches that the first step drops
    else:
        s["k"], s["v"] = _pool(g, case, case["layers"])
        pages, live, moves, slots = case["pages"], case["live"], case["moves"], case["slots"]
        low = torch.randperm(live, generator=g, device=DEVICE)[moves:]
        high = live + torch.randperm(pages - live, generator=g, device=DEVICE)[:moves]
        ids = torch.cat([low, high])[torch.randperm(live, generator=g, device=DEVICE)]
        width = -(-live // slots)
        table = torch.full((slots * width,), -1, dtype=torch.int32, device=DEVICE)
        table[:live] = ids.to(torch.int32)
        s["first_table"] = table.view(slots, width)
        s["first_refs"] = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
        s["first_refs"][ids] = 1
        s["table"], s["refs"] = s["first_table"].clone(), s["first_refs"].clone()
        s["lengths"] = (s["table"] >= 0).sum(1).to(torch.int32) * case["page"]
    if own and "table" in s:
        s["cache"] = _cache(case, s, s.get("refs"))
    return s


# ------------------------------------------------------------------- one pass

def run(s):
    case, op = s["case"], s["op"]
    if own:
        return _run_own(case, op, s)
    if op == "rotary":
        sign = -1.0 if case["inverse"] else 1.0
        return {"q": _rotate(case, s, s["q"], s["positions"], sign),
                "k": _rotate(case, s, s["new_k"], s["positions"], sign)}
    if op == "append":
        return _append(case, s)
    if op == "token":
        return {"out": _attend_paged(case, s, torch.arange(case["n"], device=DEVICE)[:, None], 1)}
    if op == "window":
        return {"out": _window(case, s)}
    if op == "fork":
        return _fork(s)
    return _compact(case, s)


def _run_own(case, op, s):
    if op == "rotary":
        q, k = s["rotary"].apply(s["q"], s["new_k"], positions=s["positions"],
                                 inverse=case["inverse"])
        return {"q": q, "k": k}
    if op == "append":
        q = s["cache"].append(s["new_k"], s["new_v"], starts=s["starts"], max_new=s["longest"],
                              rotary=s["rotary"], q=s["q"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if op == "token":
        return {"out": s["cache"].attend(s["q"], scale=s["scale"], window=case["window"] or None,
                                         sinks=case["sinks"], max_length=s["longest"])}
    if op == "window" and case["page"]:
        return {"out": s["cache"].attend(s["q"], starts=s["starts"], max_new=s["longest"],
                                         scale=s["scale"], window=case["window"],
                                         sinks=case["sinks"], max_length=s["longest"])}
    if op == "window":
        from vectorstorekit_amd import window_attention

        return {"out": window_attention(_context(), s["q"], s["k"], s["v"], starts=s["starts"],
                                        max_length=s["longest"], scale=s["scale"],
                                        window=case["window"], sinks=case["sinks"])}
    if op == "fork":
        s["cache"].fork(s["parents"], s["children"])
        return {"k": s["k"], "v": s["v"], "table": s["table"], "lengths": s["lengths"],
                "refs": s["refs"]}
    s["table"].copy_(s["first_table"])
    s["refs"].copy_(s["first_refs"])
    live = s["cache"].compact()
    return {"k": s["k"], "v": s["v"], "table": s["table"], "refs": s["refs"], "live": live}


def _rotate(case, s, x, positions, sign=1.0):
    """Each rotated pair (a, b) to (a cos - b sin, a sin + b cos)."""
    r = case["rotated"]
    c, n = s["cos"][positions.long()][:, None], sign * s["sin"][positions.long()][:, None]
    y = x.float()
    turned, rest = y[..., :r], y[..., r:]
    if case["layout"] == "half":
        a, b = turned[..., :r // 2], turned[..., r // 2:]
        turned = torch.cat([a * c - b * n, a * n + b * c], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _places(s):
    """For each new token: its sequence and its position there.  A
    sequence's new tokens are its last ones."""
    starts = s["starts"].long()
    tokens = torch.arange(s["q"].shape[0], device=DEVICE)
    seq = torch.bucketize(tokens, starts[1:], right=True)
    return seq, s["lengths"].long()[seq] - starts[seq + 1] + tokens


def _append(case, s):
    seq, pos = _places(s)
    page = s["table"].long()[seq, pos // case["page"]]
    s["k"][page, pos % case["page"]] = _rotate(case, s, s["new_k"], pos)
    s["v"][page, pos % case["page"]] = s["new_v"]
    return {"q": _rotate(case, s, s["q"], pos), "k": s["k"], "v": s["v"]}


def _softmax_sum(case, q, k, v, qpos, lengths, scale):
    """q: n x t x heads x dim, k and v: n x l x kv_heads x dim, qpos: n x t
    positions of the queries; all in 32 bits."""
    n, t, heads, d = q.shape
    l, kv = k.shape[1], k.shape[2]
    q = (q * scale).view(n, t, kv, heads // kv, d).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(q.reshape(n * kv, -1, d),
                          k.permute(0, 2, 3, 1).reshape(n * kv, d, l)).view(n, kv, -1, t, l)
    j = torch.arange(l, device=DEVICE)
    seen = (j <= qpos[..., None]) & (j < lengths[:, None, None])
    if case["window"]:
        seen &= (j > qpos[..., None] - case["window"]) | (j < case["sinks"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min_(-3e38)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(n * kv, -1, l),
                       v.permute(0, 2, 1, 3).reshape(n * kv, l, d)).view(n, kv, -1, t, d)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(n, t, heads, d)


def _attend_paged(case, s, rows, t):
    """rows: n x t, the queries' places in q."""
    n, width = s["table"].shape
    ids = s["table"].clamp(min=0).long()
    k, v = (x[ids].view(n, width * case["page"], case["kv_heads"], case["dim"]).float()
            for x in (s["k"], s["v"]))
    qpos = s["lengths"][:, None] - t + torch.arange(t, device=DEVICE)
    return _softmax_sum(case, s["q"][rows].float(), k, v, qpos, s["lengths"],
                        s["scale"]).flatten(0, 1).to(s["q"].dtype)


def _window(case, s):
    """Prompts whose tokens are the whole sequence: padded to the longest."""
    t, tokens = s["longest"], s["q"].shape[0]
    places = s["starts"][:-1, None].long() + torch.arange(t, device=DEVICE)
    real = torch.arange(t, device=DEVICE) < s["lengths"][:, None]
    places = places.clamp(max=tokens - 1)
    if case["page"]:
        n, width = s["table"].shape
        ids = s["table"].clamp(min=0).long()
        k, v = (x[ids].view(n, width * case["page"], case["kv_heads"], case["dim"]).float()
                for x in (s["k"], s["v"]))
    else:
        k, v = s["k"][places].float(), s["v"][places].float()
    qpos = torch.arange(t, device=DEVICE).expand(case["n"], t)
    out = _softmax_sum(case, s["q"][places].float(), k, v, qpos, s["lengths"], s["scale"])
    return out[real].to(s["q"].dtype)


def _fork(s):
    """What the children held is released; each then shares its parent's
    whole pages and gets a copy of the rows of a last page that is not full,
    in the lowest free page (in the children's order)."""
    table, refs, lengths = s["table"], s["refs"], s["lengths"]
    parents, children = s["parents"].long(), s["children"].long()
    page, width = s["k"].shape[-3], table.shape[1]
    slot = torch.arange(width, device=DEVICE)
    old = table[children]
    refs.index_add_(0, old.clamp(min=0).flatten().long(), -(old >= 0).flatten().int())
    full, fill = lengths[parents] // page, lengths[parents] % page
    new = torch.where(slot < full[:, None], table[parents], -1)
    refs.index_add_(0, new.clamp(min=0).flatten().long(), (new >= 0).flatten().int())
    split = fill > 0
    free = torch.sort((refs > 0).to(torch.uint8), stable=True).indices
    rank = (torch.cumsum(split, 0) - 1).clamp(min=0)
    at = torch.where(split, free[rank], refs.shape[0])
    refs.index_add_(0, at[split], torch.ones_like(at[split], dtype=torch.int32))
    last = table[parents, full.clamp(max=width - 1).long()].long()
    new = torch.where((slot == full[:, None]) & split[:, None], at[:, None].int(), new)
    src, dst = last[split], at[split]
    rows = (torch.arange(page, device=DEVICE) < fill[split][:, None])[None, :, :, None, None]
    for pool in (s["k"], s["v"]):
        pool[:, dst] = torch.where(rows, pool[:, src], pool[:, dst])
    table[children], lengths[children] = new, lengths[parents]
    return {"k": s["k"], "v": s["v"], "table": table, "lengths": lengths, "refs": refs}


def _compact(case, s):
    """With m pages in use, those numbered m and above move, in order, to
    the free ones below m."""
    table, refs = s["table"].copy_(s["first_table"]), s["refs"].copy_(s["first_refs"])
    used = refs > 0
    live = used.sum()
    ids = torch.arange(refs.shape[0], device=DEVICE)
    dst, src = ids[~used & (ids < live)], ids[used & (ids >= live)]
    for pool in (s["k"], s["v"]):
        pool[:, dst] = pool[:, src]
    place = ids.clone()
    place[src] = dst
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()].int(), -1))
    refs[dst] = refs[src]
    refs[src] = 0
    return {"k": s["k"], "v": s["v"], "table": table, "refs": refs, "live": live.to(torch.int32)}


# ------------------------------------------------- what a pass cannot do without

def _visible(case, length, new):
    """Pairs of a query and a key it sees, for the last ``new`` tokens of a
    sequence, and the keys that any of them sees."""
    i = np.arange(length - new, length, dtype=np.int64)
    w, sinks = case["window"] or length, case["sinks"]
    pairs = np.minimum(i + 1, w) + np.clip(i + 1 - w, 0, sinks)
    first = max(0, length - new - w + 1)
    return int(pairs.sum()), length - first + min(first, sinks)


def work(case):
    op, size = case["op"], TYPES[case["type"]].itemsize
    if op in ("rotary", "append"):
        tokens = case["tokens"] if op == "rotary" else sum(_lengths(case))
        values = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        turned = tokens * (case["heads"] + case["kv_heads"]) * case["rotated"]
        if op == "append":
            values += tokens * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * values * size + 4 * tokens, "flops": 3 * turned}
    if op in ("token", "window"):
        pairs = keys = 0
        lengths = _lengths(case)
        for x in lengths:
            p, k = _visible(case, x, 1 if op == "token" else x)
            pairs, keys = pairs + p, keys + k
        tokens = case["n"] if op == "token" else sum(lengths)
        return {"bytes": size * case["dim"] * 2 * (keys * case["kv_heads"]
                                                   + tokens * case["heads"]),
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * size
    if op == "fork":
        # the parents are drawn by the seed: half a page a branch on average
        return {"bytes": 2 * row * case["n"] * case["page"] // 2 + 8 * case["pages"], "flops": 0}
    return {"bytes": 2 * row * case["page"] * case["moves"] + 8 * (case["pages"] + case["live"]),
            "flops": 0}


# --------------------------------------------------------- the definition, 64 bits

def _turned(case, x, positions, sign=1.0):
    inv, amplitude = _frequencies(case)
    r, y = case["rotated"], x.double().clone()
    angle = positions.double()[:, None, None] * torch.from_numpy(inv).to(DEVICE)
    first = (slice(0, r // 2) if case["layout"] == "half" else slice(0, r, 2))
    second = (slice(r // 2, r) if case["layout"] == "half" else slice(1, r, 2))
    z = torch.complex(y[..., first], y[..., second])
    z = z * torch.polar(torch.full_like(angle, amplitude), sign * angle)
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _sequence(case, s, b, length):
    """Keys and values of one sequence in 64 bits, kv_heads x length x dim."""
    if case["page"]:
        ids = s["table"][b, :-(-length // case["page"])].long()
        k, v = (s[x][ids].flatten(0, 1)[:length] for x in "kv")
    else:
        at = int(s["starts"][b])
        k, v = (s[x][at:at + length] for x in "kv")
    return k.double().transpose(0, 1).contiguous(), v.double().transpose(0, 1).contiguous()


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "rotary":
        sign = -1.0 if case["inverse"] else 1.0
        return {"q": _turned(case, s["q"], s["positions"], sign),
                "k": _turned(case, s["new_k"], s["positions"], sign)}
    if op == "append":
        k, v, out = s["k"].double(), s["v"].double(), []
        for b, x in enumerate(_lengths(case)):
            at, pos = int(s["starts"][b]), torch.arange(x, 2 * x, device=DEVICE)
            page, row = s["table"][b].long()[pos // case["page"]], pos % case["page"]
            k[page, row] = _turned(case, s["new_k"][at:at + x], pos)
            v[page, row] = s["new_v"][at:at + x].double()
            out.append(_turned(case, s["q"][at:at + x], pos))
        return {"q": torch.cat(out), "k": k, "v": v}
    if op not in ("token", "window"):
        return None
    out, heads, group = [], case["heads"], case["heads"] // case["kv_heads"]
    for b, length in enumerate(_lengths(case)):
        new = 1 if op == "token" else length
        at = int(s["starts"][b])
        q = s["q"][at:at + new].double()
        k, v = _sequence(case, s, b, length)
        done = torch.empty(new, heads, case["dim"], dtype=torch.float64, device=DEVICE)
        for t0 in range(0, new, 1024):
            t1 = min(t0 + 1024, new)
            i = torch.arange(length - new + t0, length - new + t1, device=DEVICE)[:, None]
            j = torch.arange(length, device=DEVICE)[None]
            seen = j <= i
            if case["window"]:
                seen = seen & ((i - j < case["window"]) | (j < case["sinks"]))
            for h in range(heads):
                x = q[t0:t1, h] @ k[h // group].T * case["dim"] ** -0.5
                p = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
                done[t0:t1, h] = p @ v[h // group]
        out.append(done)
    return {"out": torch.cat(out)}
