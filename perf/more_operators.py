"""Performance cases of answering many questions over the same documents: what
is timed, on which inputs, and what the results are.

The operators are the decoder's projections in 8 bits (scales for each token
and each channel), cross attention to encoded documents of another length, and
attention over the paged cache for branches that share a long prefix.

``listed`` names the cases, ``draw`` makes others of the same ranges,
``prepare`` makes what a program holds before the call and ``run`` makes the
call: with ``own`` through the package's public classes, without it as
elementary torch operations in 32 bits (64 for the sums of integers, which 32
do not hold), rounded once at the end.  ``work`` states the bytes and
operations a call cannot do without and ``exact`` evaluates the definition in
64 bits.
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
        # one conversation's next token through a projection: latency
        {"name": "linear_token", "op": "linear", "tokens": 1, "inputs": 4096, "outputs": 4096,
         "bias": False, "type": "bf16"},
        # a decoding step of a serving batch: the weights are what is read
        {"name": "linear_step", "op": "linear", "tokens": 64, "inputs": 4096, "outputs": 12288,
         "bias": True, "type": "bf16"},
        # a small head of odd sizes, 32-bit activations
        {"name": "linear_odd", "op": "linear", "tokens": 777, "inputs": 1000, "outputs": 1777,
         "bias": True, "type": "f32"},
        # long prompts: the matrix cores are what is used
        {"name": "linear_prompt", "op": "linear", "tokens": 16384, "inputs": 4096,
         "outputs": 12288, "bias": False, "type": "bf16"},
        # one token against one short document: latency
        {"name": "cross_token", "op": "cross", "n": 1, "new": 1, "sets": 1, "longest": 300,
         "padded": False, "heads": 8, "kv_heads": 8, "dim": 64, "type": "f16"},
        # a decoding step of a batch padded to its longest document, a few
        # candidates each
        {"name": "cross_step", "op": "cross", "n": 64, "new": 4, "sets": 64, "longest": 4096,
         "padded": True, "heads": 16, "kv_heads": 16, "dim": 64, "type": "bf16"},
        # ragged prompts against the documents found for them
        {"name": "cross_prompt", "op": "cross", "n": 8, "new": 2048, "sets": 8, "longest": 8192,
         "padded": False, "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16"},
        # several questions about the same few documents, in 32 bits
        {"name": "cross_same", "op": "cross", "n": 7, "new": 500, "sets": 3, "longest": 3001,
         "padded": False, "heads": 20, "kv_heads": 5, "dim": 80, "type": "f32"},
        # a few branches of a short retrieved context: latency
        {"name": "shared_few", "op": "shared", "groups": 1, "members": 4, "prefix": 512,
         "tail": 40, "new": 1, "page": 16, "heads": 8, "kv_heads": 2, "dim": 64, "type": "bf16"},
        # many answers over one long set of documents
        {"name": "shared_batch", "op": "shared", "groups": 1, "members": 64, "prefix": 32768,
         "tail": 512, "new": 1, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "bf16"},
        # a serving batch: several documents, some with one reader only
        {"name": "shared_groups", "op": "shared", "groups": 12, "members": 16, "prefix": 8000,
         "tail": 2000, "new": 1, "page": 16, "heads": 28, "kv_heads": 4, "dim": 128,
         "type": "f16"},
        # several new tokens a branch, every head with keys of its own, 32 bits
        {"name": "shared_drafts", "op": "shared", "groups": 6, "members": 10, "prefix": 4000,
         "tail": 300, "new": 9, "page": 32, "heads": 16, "kv_heads": 16, "dim": 96,
         "type": "f32"},
    ]


#: heads, heads of keys and values, and their dimension
HEADS = [(32, 8, 128), (16, 16, 64), (8, 1, 256), (12, 12, 96), (28, 4, 128), (20, 5, 80),
         (64, 8, 128), (9, 3, 64)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(["linear", "cross", "shared"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "linear":
        inputs, outputs = (_log(rng, 64, 12288) for _ in range(2))
        if rng.random() < 0.5:  # (widths of models are round, others need not be)
            inputs, outputs = (-(-x // 64) * 64 for x in (inputs, outputs))
        tokens = _log(rng, 1, min(16384, 16384 * 4096 * 6144 // (inputs * outputs)))
        return {"op": op, "tokens": tokens, "inputs": inputs, "outputs": outputs,
                "bias": rng.random() < 0.5, "type": kind}
    heads, kv_heads, dim = rng.choice(HEADS)
    base = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "type": kind}
    slow = 8 if kind == "f32" else 1
    if op == "cross":
        n = _log(rng, 1, 64)
        # the largest: 8 x 2048 queries of 32 heads of 128, 8192 keys; and 512 MiB of keys
        most = max(1, 8 * 2048 * 32 * 128 // (slow * n * heads * dim))
        new = rng.choice([1, _log(rng, 1, min(8, most)), _log(rng, 1, min(2048, most))])
        pairs = 8 * 2048 * 8192 * 32 * 128 // (2 * slow)
        held = (1 << 29) // (4 * kv_heads * dim)
        sets = rng.choice([n, n, _log(rng, 1, n)])
        longest = _log(rng, 1, max(1, min(16384, pairs // (n * new * heads * dim), held // sets)))
        return {**base, "n": n, "new": new, "sets": sets, "longest": longest,
                "padded": rng.random() < 0.4}
    groups, members = _log(rng, 1, 12), _log(rng, 1, 64)
    members = min(members, max(1, 128 // groups))
    page = rng.choice([16, 32, 64, 128])
    new = rng.choice([1, 1, _log(rng, 2, 12)])
    tail = _log(rng, new, 2000)
    room = (1 << 29) // (4 * kv_heads * dim) - groups * members * (tail + page)
    if room < groups * page:
        groups, members, room = 1, 4, 32768
    rows = groups * members * new * heads * dim
    prefix = _log(rng, 1, max(page, min(32768, room // groups, (1 << 36) // (slow * rows))))
    return {**base, "groups": groups, "members": members, "prefix": prefix, "tail": tail,
            "new": new, "page": page}


# ------------------------------------------------------- what the cases stand on
# Lengths are a case's own, whatever the seed, so that its work is known.

def _ragged(rng, top, count, least):
    """Ragged lengths, the first the longest."""
    return [top] + [least + int((top - least) * rng.random() ** 1.5) for _ in range(count - 1)]


def _cross_lengths(case):
    """New tokens of each sequence, keys of each set, each sequence's set."""
    rng = random.Random(case["longest"] * 7919 + case["n"])
    n, sets = case["n"], case["sets"]
    new = [case["new"]] * n if case["padded"] else _ragged(rng, case["new"], n, 1)
    keys = _ragged(rng, case["longest"], sets, 0 if sets > 2 else 1)
    which = list(range(n)) if sets == n else [0] + [rng.randrange(sets) for _ in range(n - 1)]
    return new, keys, which


def _shared_lengths(case):
    """For each group: keys shared (whole pages), and for each of its members
    the keys of its own and, of those, the new tokens."""
    rng = random.Random(case["prefix"] * 7919 + case["members"])
    page = case["page"]
    prefixes = [p // page * page for p in _ragged(rng, case["prefix"], case["groups"], 1)]
    sizes = _ragged(rng, case["members"], case["groups"], 1)
    out = []
    for p, size in zip(prefixes, sizes):
        tails = _ragged(rng, case["tail"], size, 1)
        new = [min(t, case["new"] if i == 0 else rng.randint(1, case["new"]))
               for i, t in enumerate(tails)]
        out.append((p, tails, new))
    return out


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _projected(g, *shape, dtype):
    """Activations, queries or keys as projections make them: some channels
    stand out."""
    x = torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)
    loud = 1.0 + 2.0 * (torch.rand(shape[-1], generator=g, device=DEVICE) < 0.05)
    return x.mul_(loud).to(dtype)


def _starts(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g, op, t = _generator(seed), case["op"], TYPES[case["type"]]
    s = {"case": case, "op": op}
    if op == "linear":
        m, k, n = case["tokens"], case["inputs"], case["outputs"]
        s["x"] = _projected(g, m, k, dtype=t)
        # weights as they are kept: codes and a scale for each channel
        s["codes"] = (torch.randn(n, k, generator=g, device=DEVICE) * 40).round_() \
            .clamp_(-127, 127).to(torch.int8)
        s["scales"] = (0.5 + torch.rand(n, generator=g, device=DEVICE)) * k ** -0.5 / 40
        s["bias"] = _normal(g, n, dtype=torch.float32) if case["bias"] else None
        if own:
            from vectorstorekit_amd import Int8Linear

            s["layer"] = Int8Linear.over(_context(), s["codes"], s["scales"], s["bias"])
        return s
    s["scale"] = case["dim"] ** -0.5
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if op == "cross":
        new, keys, which = _cross_lengths(case)
        s["q"] = _projected(g, sum(new), heads, dim, dtype=t)
        s["starts"] = None if case["new"] == 1 else _starts(new)
        s["sets"] = None if case["sets"] == case["n"] else \
            torch.tensor(which, dtype=torch.int32, device=DEVICE)
        shape = ((case["sets"], case["longest"]) if case["padded"] else (sum(keys),))
        s["k"] = _projected(g, *shape, kv_heads, dim, dtype=t)
        s["v"] = _normal(g, *shape, kv_heads, dim, dtype=t)
        if case["padded"]:
            s["lengths"] = torch.tensor(keys, dtype=torch.int32, device=DEVICE)
        else:
            s["k_starts"] = _starts(keys)
        return s
    page, groups = case["page"], _shared_lengths(case)
    # pages from all over the pool; a group's members share the prefix's
    width = max(p // page + -(-max(tails) // page) for p, tails, _ in groups)
    pages = sum(p // page + sum(-(-x // page) for x in tails) for p, tails, _ in groups) + 3
    ids = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    rows, at = [], 0
    for p, tails, _ in groups:
        first, at = np.arange(at, at + p // page), at + p // page
        for x in tails:
            u = -(-x // page)
            row = np.concatenate([first, np.arange(at, at + u)])
            rows.append(np.pad(row, (0, width - len(row)), constant_values=-1))
            at += u
    table = torch.from_numpy(np.stack(rows)).to(DEVICE)
    s["table"] = torch.where(table >= 0, ids[table.clamp(min=0)], -1).to(torch.int32)
    s["lengths"] = torch.tensor([p + x for p, tails, _ in groups for x in tails],
                                dtype=torch.int32, device=DEVICE)
    shape = (pages, page, kv_heads, dim)
    s["k"], s["v"] = _projected(g, *shape, dtype=t), _normal(g, *shape, dtype=t)
    new = [x for _, _, counts in groups for x in counts]
    s["q"] = _projected(g, sum(new), heads, dim, dtype=t)
    s["starts"] = None if case["new"] == 1 else _starts(new)
    if own:
        from vectorstorekit_amd import PagedKVCache

        s["cache"] = PagedKVCache.over(_context(), s["k"], s["v"], s["table"], s["lengths"])
        # made when the branches are forked, used by every layer and step
        offsets = [0] + list(np.cumsum([len(tails) for _, tails, _ in groups]))
        s["plan"] = s["cache"].share(offsets, prefix=case["prefix"])
    return s


# ------------------------------------------------------------------- one pass

def run(s):
    case, op = s["case"], s["op"]
    if own:
        return _run_own(case, op, s)
    if op == "linear":
        return {"out": _linear(s)}
    if op == "cross":
        return {"out": _cross(case, s)}
    return {"out": _shared(case, s)}


def _run_own(case, op, s):
    if op == "linear":
        return {"out": s["layer"](s["x"])}
    if op == "cross":
        from vectorstorekit_amd import cross_attention

        keys = ({"k_lengths": s["lengths"]} if case["padded"] else
                {"k_starts": s["k_starts"], "max_keys": case["longest"]})
        return {"out": cross_attention(_context(), s["q"], s["k"], s["v"], starts=s["starts"],
                                       sets=s["sets"], max_length=case["new"], scale=s["scale"],
                                       **keys)}
    return {"out": s["cache"].attend(s["q"], starts=s["starts"], max_new=case["new"],
                                     scale=s["scale"], shared=s["plan"],
                                     max_length=case["prefix"] + case["tail"])}


def _codes(x):
    """Each row's codes, whole numbers of at most 127, and its scale.  (Rows
    of tiny numbers are first made larger by a power of two, so that 127 over
    their largest is finite.)"""
    y = x.float()
    top = y.abs().amax(-1, keepdim=True)
    up = torch.where(top < 2.0 ** -100, 2.0 ** 100, 1.0)
    most = torch.full_like(top, 127.0)
    inverse = torch.where(top > 0, torch.div(most, top * up), 0.0)
    return torch.round(y * up * inverse).clamp_(-127, 127), torch.div(top, most)


def _linear(s):
    codes, scales = _codes(s["x"])
    sums = torch.matmul(codes.double(), s["codes"].double().T)
    out = sums.float() * scales * s["scales"]
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(s["x"].dtype)


def _softmax_parts(scores):
    """(weights, their sums, the maxima) along the last dimension, in place."""
    top = scores.amax(-1, keepdim=True).clamp_min_(-3e38)
    scores.sub_(top).exp_()
    return scores, scores.sum(-1, keepdim=True), top


def _cross(case, s):
    new, keys, which = _cross_lengths(case)
    heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["padded"] and s["sets"] is None:
        n, t, l = case["n"], case["new"], case["longest"]
        q = (s["q"].float() * s["scale"]).view(n, t, kv, heads // kv, d).permute(0, 2, 3, 1, 4)
        k = s["k"].float().permute(0, 2, 3, 1).reshape(n * kv, d, l)
        scores = torch.matmul(q.reshape(n * kv, -1, d), k).view(n, kv, -1, l)
        seen = torch.arange(l, device=DEVICE) < s["lengths"][:, None]
        scores.masked_fill_(~seen[:, None, None], -math.inf)
        w, total, _ = _softmax_parts(scores)
        v = s["v"].float().permute(0, 2, 1, 3).reshape(n * kv, l, d)
        out = torch.matmul(w.view(n * kv, -1, l), v).view(n, kv, -1, d)
        out = torch.where(total > 0, out / total, 0.0).view(n, kv, heads // kv, t, d)
        return out.permute(0, 3, 1, 2, 4).reshape(n * t, heads, d).to(s["q"].dtype)
    out, at = torch.zeros_like(s["q"]), 0
    offsets = [0] + list(np.cumsum(keys))
    for t, z in zip(new, which):
        l = keys[z]
        if l:
            if case["padded"]:
                k, v = s["k"][z, :l], s["v"][z, :l]
            else:
                k, v = (s[x][offsets[z]:offsets[z] + l] for x in "kv")
            q = (s["q"][at:at + t].float() * s["scale"]).view(t, kv, heads // kv, d)
            q = q.permute(1, 2, 0, 3).reshape(kv, -1, d)
            w, total, _ = _softmax_parts(torch.matmul(q, k.float().permute(1, 2, 0).contiguous()))
            y = torch.matmul(w, v.float().transpose(0, 1).contiguous()) / total
            out[at:at + t] = y.view(kv, heads // kv, t, d).permute(2, 0, 1, 3).reshape(t, heads, d)
        at += t
    return out


def _shared(case, s):
    """The prefix's scores once for a group's rows; the members' own keys
    padded to the longest; both under one softmax."""
    page, kv, d = case["page"], case["kv_heads"], case["dim"]
    group = case["heads"] // kv
    out, at, slot = torch.empty_like(s["q"]), 0, 0
    for p, tails, new in _shared_lengths(case):
        m, t = len(tails), max(new)
        lengths = torch.tensor(tails, device=DEVICE)
        counts = torch.tensor(new, device=DEVICE)
        first = at + torch.cumsum(counts, 0) - counts
        i = torch.arange(t, device=DEVICE)
        places = (first[:, None] + i).clamp(max=s["q"].shape[0] - 1)
        q = (s["q"][places].float() * s["scale"]).view(m, t, kv, group, d)
        q = q.permute(2, 0, 3, 1, 4).contiguous()  # kv, member, head, token, d
        ids = s["table"][slot, :p // page].long()
        pk, pv = (s[x][ids].flatten(0, 1).float().transpose(0, 1).contiguous() for x in "kv")
        ids = s["table"][slot:slot + m, p // page:].clamp(min=0).long()
        ids = ids[:, :-(-max(tails) // page)]
        tk, tv = (s[x][ids].flatten(1, 2).float() for x in "kv")  # member, key, kv, d
        tk = tk.permute(2, 0, 3, 1).contiguous()  # kv, member, d, key
        tv = tv.permute(2, 0, 1, 3).contiguous()  # kv, member, key, d
        a = torch.matmul(q.view(kv, -1, d), pk.transpose(1, 2).contiguous()) \
            .view(kv, m, group, t, p)
        b = torch.matmul(q.view(kv, m, -1, d), tk).view(kv, m, group, t, -1)
        j = torch.arange(b.shape[-1], device=DEVICE)
        seen = j <= (lengths - counts)[:, None, None] + i[:, None]  # member, token, key
        b.masked_fill_(~seen[None, :, None], -math.inf)
        w, total, _ = _softmax_parts(torch.cat([a, b], -1))
        y = torch.matmul(w[..., :p].reshape(kv, m * group * t, p), pv).view(kv, m, group, t, d)
        y = y + torch.matmul(w[..., p:].reshape(kv, m, group * t, -1), tv) \
            .view(kv, m, group, t, d)
        y = (y / total).permute(1, 3, 0, 2, 4).reshape(m, t, kv * group, d)
        out[at:at + sum(new)] = y[i < counts[:, None]].to(out.dtype)
        at, slot = at + sum(new), slot + m
    return out


# ------------------------------------------------- what a pass cannot do without

def work(case):
    size = TYPES[case["type"]].itemsize
    if case["op"] == "linear":
        m, k, n = case["tokens"], case["inputs"], case["outputs"]
        return {"bytes": size * m * (k + n) + n * k + (8 if case["bias"] else 4) * n,
                "flops": 2 * m * n * k}
    heads, row = case["heads"] * case["dim"], 2 * case["kv_heads"] * case["dim"] * size
    if case["op"] == "cross":
        new, keys, which = _cross_lengths(case)
        used = sum(keys[z] for z in set(which))
        pairs = sum(t * keys[z] for t, z in zip(new, which))
        return {"bytes": row * used + 2 * size * heads * sum(new), "flops": 4 * heads * pairs}
    pairs = keys = tokens = 0
    for p, tails, new in _shared_lengths(case):
        keys += p + sum(tails)
        tokens += sum(new)
        pairs += sum(t * (p + x) - t * (t - 1) // 2 for x, t in zip(tails, new))
    return {"bytes": row * keys + 2 * size * heads * tokens, "flops": 4 * heads * pairs}


# --------------------------------------------------------- the definition, 64 bits

def _attended(q, k, v, scale, pos):
    """q: t x heads x d, k and v: l x kv x d; query i sees the keys up to
    pos[i]."""
    t, heads, d = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(t, heads, d, dtype=torch.float64, device=DEVICE)
    if not k.shape[0]:
        return out
    hidden = torch.arange(k.shape[0], device=DEVICE)[None] > pos[:, None]
    for h in range(heads):
        kh, vh = k[:, h // group].double(), v[:, h // group].double()
        for a in range(0, t, 1024):
            x = q[a:a + 1024, h].double() @ kh.T * scale
            w = torch.softmax(x.masked_fill_(hidden[a:a + 1024], -math.inf), -1)
            out[a:a + 1024, h] = w @ vh
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "linear":
        # (the codes are whole numbers by definition: quotients of 32 bits, rounded)
        x = s["x"].float()
        top = x.abs().max(1, keepdim=True).values
        shift = 100 * (top < 2.0 ** -100)
        inverse = torch.where(top > 0, torch.full_like(top, 127) / torch.ldexp(top, shift), top)
        codes = torch.round(torch.ldexp(x, shift) * inverse).double().clamp(-127, 127)
        weights = s["codes"].double() * s["scales"].double()[:, None]
        out = (codes * (top.double() / 127)) @ weights.T
        return {"out": out if s["bias"] is None else out + s["bias"].double()}
    at, parts = 0, []
    if op == "cross":
        new, keys, which = _cross_lengths(case)
        offsets = np.cumsum([0] + keys)
        for t, z in zip(new, which):
            lo = offsets[z]
            k, v = (s[x][z, :keys[z]] if case["padded"] else s[x][lo:lo + keys[z]] for x in "kv")
            see = torch.full((t,), keys[z], device=DEVICE)
            parts.append(_attended(s["q"][at:at + t], k, v, s["scale"], see))
            at += t
        return {"out": torch.cat(parts)}
    slot = 0
    for p, tails, new in _shared_lengths(case):
        for x, t in zip(tails, new):
            ids = s["table"][slot, :-(-(p + x) // case["page"])].long()
            k, v = (s[y][ids].flatten(0, 1)[:p + x] for y in "kv")
            pos = torch.arange(p + x - t, p + x, device=DEVICE)
            parts.append(_attended(s["q"][at:at + t], k, v, s["scale"], pos))
            at, slot = at + t, slot + 1
    return {"out": torch.cat(parts)}
