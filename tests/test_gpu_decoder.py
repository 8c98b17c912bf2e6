"""A decoder's step over retrieved documents with 8-bit projections, branches
that share their context and cross attention to an encoder's states, each call
against 64 bits on the inputs that it had, and the whole captured and replayed.

The tolerances of each call are those of its own tests."""
import importlib.util
import math
import os

import pytest
import torch

from test_gpu_linear import BF, DEV, F32, check, expected, gen, normal
from test_gpu_shared import attended, check_shared, ints

pytestmark = pytest.mark.gpu

HEADS, KV, D, WIDTH = 8, 2, 64, 512


class Block:
    """Self attention over branches, cross attention over documents, a layer."""

    def __init__(self, ctx, g, dtype):
        from vectorstorekit_amd import Int8Linear, RotaryEmbedding

        def layer(outputs, inputs=WIDTH):
            return Int8Linear(ctx, normal(g, outputs, inputs, dtype=dtype) * inputs ** -0.5,
                              normal(g, outputs))

        self.ctx, self.rotary = ctx, RotaryEmbedding(ctx, D)
        self.qkv, self.out = layer((HEADS + 2 * KV) * D), layer(WIDTH)
        self.q, self.kv, self.last = layer(HEADS * D), layer(2 * KV * D), layer(WIDTH)
        self.head = layer(1000)

    def states(self, x):
        """Keys and values of documents' states (sets x length x WIDTH)."""
        return self.kv(x).unflatten(-1, (2, KV, D)).unbind(2)

    def heads_of(self, x):
        return self.qkv(x).unflatten(-1, (-1, D)).split([HEADS, KV, KV], 1)

    def step(self, x, cache, plan, documents, lengths, sets):
        """Every call's inputs and output."""
        from vectorstorekit_amd import cross_attention

        calls = {}
        q, k, v = self.heads_of(x)
        q = cache.append(k, v, seqs=plan.seqs, rotary=self.rotary, q=q)
        calls["self"] = q, cache.attend(q, shared=plan)
        y = calls["self"][1].flatten(1)
        calls["out"] = y, self.out(y)
        x = x + calls["out"][1]
        calls["q"] = x, self.q(x)
        q = calls["q"][1].unflatten(1, (HEADS, D))
        calls["cross"] = q, cross_attention(self.ctx, q, *documents, k_lengths=lengths, sets=sets)
        y = calls["cross"][1].flatten(1)
        calls["last"] = y, self.last(y)
        x = x + calls["last"][1]
        calls["head"] = x, self.head(x, dtype=F32)
        return calls


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("branches,context", [(4, 150), (40, 1000)])
def test_steps(ctx, dtype, branches, context):
    from vectorstorekit_amd import PagedKVCache

    g = gen(branches)
    block = Block(ctx, g, dtype)
    cache = PagedKVCache(ctx, pages=400, page_size=16, kv_heads=KV, head_dim=D,
                         slots=branches + 1, width=80, dtype=dtype)
    # the context, and branches of it
    cache.reserve([0], [context])
    _, k, v = block.heads_of(normal(g, context, WIDTH, dtype=dtype))
    cache.append(k, v, starts=[0, context], seqs=[0], rotary=block.rotary)
    slots = ints(range(1, branches + 1))
    cache.fork(torch.zeros_like(slots), slots)
    plan = cache.share([0, branches], seqs=slots)
    assert plan.prefix.tolist() == [context // 16 * 16] * branches
    # the documents found, of which each branch looks at one
    documents = block.states(normal(g, 3, 90, WIDTH, dtype=dtype))
    lengths, sets = ints([90, 17, 64]), ints([i % 3 for i in range(branches)])
    ones, x = torch.ones_like(slots), normal(g, branches, WIDTH, dtype=dtype)

    def step():
        cache.reserve(slots, ones)
        return block.step(x, cache, plan, documents, lengths, sets)

    def checked(calls):
        class One:
            k, v, table, lengths = cache.k[0], cache.v[0], cache.table, cache.lengths
            page_size = cache.page_size

        q, out = calls["self"]
        check_shared(One, slots.tolist(), q, None, out, D ** -0.5)
        q, out = calls["cross"]
        for i in range(branches):
            k, v = (y[i % 3, :int(lengths_now[i % 3])] for y in documents)
            want, _, tol = attended(q[i:i + 1], k, v, [len(k)], D ** -0.5)
            check(out[i:i + 1], want, tol)
        for name in ("out", "q", "last", "head"):
            layer, (y, out) = getattr(block, name), calls[name]
            check(out, *expected(y, layer.codes(), layer.scales, layer.bias, out.dtype))

    lengths_now = lengths.tolist()
    checked(step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls = step()
    for i in range(4):
        x.copy_(normal(g, branches, WIDTH, dtype=dtype))
        lengths.copy_(ints([90 - i, 17 + i, i]))
        lengths_now = lengths.tolist()
        graph.replay()
        torch.cuda.synchronize()
        # (what the graph left is looked at before other work, and after it)
        kept = {n: [y.clone() for y in c] for n, c in calls.items()}
        checked(kept)
        block.head(normal(g, 300, WIDTH, dtype=dtype))
    assert cache.missing() == 0
    assert cache.lengths.tolist() == [context] + [context + 5] * branches


@pytest.mark.parametrize("eight_bits", [False, True])
def test_example(capsys, eight_bits):
    """The example with its options.  Without 8-bit codes it is held to itself
    without a cache: sixteen roundings a layer of 2^-8 of a value, four layers,
    added as independent errors, are 2^-8 sqrt(64) = 0.031 of a logit's size,
    twice that for the largest of them.  (A code is a step of its row's largest
    / 127, so that roundings before it can become whole steps.)"""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "answer_over_retrieved.py")
    spec = importlib.util.spec_from_file_location("answer_over_retrieved", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    worst = example.main(branches=3, steps=6, eight_bits=eight_bits, states=True)
    assert math.isfinite(worst) and (eight_bits or worst <= 0.0625)
    assert "documents [123" in capsys.readouterr().out
