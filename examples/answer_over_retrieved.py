"""Retrieval and what a decoder does with it, on one GPU.

    python examples/answer_over_retrieved.py [--eight-bits] [--states]

A question is searched for among documents' vectors; the documents found, and
the question, are the prompt of a small decoder with random weights (rotary
positions, fewer key heads than query heads, every second layer through a
sliding window with sinks).  The prompt goes into a paged cache, the context is
forked into branches, each branch decodes a few tokens of its own, reading what
they share once for all of them, and the branches are dropped and the pool
compacted.  With ``--eight-bits`` the projections are 8-bit layers; with
``--states`` the decoder looks also at an encoder's states of the documents
found (cross attention).  What is printed last is the largest difference to the
same tokens computed without a cache.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from vectorstorekit_amd import (Context, Int8Linear, PagedKVCache, RotaryEmbedding,  # noqa: E402
                                VectorDatabase, cross_attention, window_attention)

VOCABULARY, DOCUMENTS, LENGTH = 512, 1000, 48


class Decoder:
    """Random weights; embedding in, logits out."""

    def __init__(self, ctx, layers=4, heads=8, kv_heads=2, head_dim=64, window=96, sinks=4,
                 dtype=torch.bfloat16, seed=0, eight_bits=False):
        self.ctx, self.layers, self.heads, self.kv_heads = ctx, layers, heads, kv_heads
        self.head_dim, self.window, self.sinks, self.dtype = head_dim, window, sinks, dtype
        self.rotary = RotaryEmbedding(ctx, head_dim, scaling={"type": "yarn", "factor": 4.0,
                                                              "original_length": 512})
        width = heads * head_dim
        g = torch.Generator().manual_seed(seed)

        def weights(rows, columns):
            w = torch.randn(rows, columns, generator=g) * rows ** -0.5
            return w.to(f"cuda:{ctx.device}", dtype)

        def projection(rows, columns):
            w = weights(rows, columns)
            return Int8Linear(ctx, w.T) if eight_bits else lambda x: x @ w

        self.embedding = weights(VOCABULARY, width) * VOCABULARY ** 0.5
        self.qkv = [projection(width, (heads + 2 * kv_heads) * head_dim) for _ in range(layers)]
        self.out = [projection(width, width) for _ in range(layers)]
        self.head = projection(width, VOCABULARY)
        # queries over documents' states, the states' keys and values, and the way back
        self.documents = None
        self.look = [projection(width, width) for _ in range(layers)]
        self.read = [projection(width, 2 * kv_heads * head_dim) for _ in range(layers)]
        self.back = [projection(width, width) for _ in range(layers)]

    def look_at(self, states):
        """The documents' states (documents x length x width) that the tokens
        look at from now on: their keys and values in every layer, of one set
        for each sequence to see."""
        states = torch.nn.functional.rms_norm(states, states.shape[-1:]).flatten(0, 1)
        self.documents = [y.view(1, len(states), 2, self.kv_heads, self.head_dim).unbind(2)
                          for y in (read(states) for read in self.read)]

    def seen(self, layer):
        """The window of a layer."""
        return {"window": self.window, "sinks": self.sinks} if layer % 2 else {}

    def __call__(self, tokens, attend):
        """Logits of tokens; attend(layer, q, k, v) gives the heads' outputs."""
        x = self.embedding[tokens]
        whole = torch.tensor([0, len(tokens)], dtype=torch.int32, device=tokens.device)
        one = torch.zeros(1, dtype=torch.int32, device=tokens.device)
        for i in range(self.layers):
            y = self.qkv[i](torch.nn.functional.rms_norm(x, x.shape[-1:]))
            y = y.view(len(tokens), -1, self.head_dim)
            q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
            x = x + self.out[i](attend(i, q, k, v).flatten(1))
            if self.documents is not None:
                y = self.look[i](torch.nn.functional.rms_norm(x, x.shape[-1:]))
                q = y.view(len(tokens), self.heads, self.head_dim)
                y = cross_attention(self.ctx, q, *self.documents[i], starts=whole, sets=one)
                x = x + self.back[i](y.flatten(1))
        return self.head(torch.nn.functional.rms_norm(x, x.shape[-1:]))

    def over_cache(self, tokens, cache, seqs, starts=None, max_new=None, shared=None):
        """The tokens are the last ones of the sequences in slots ``seqs``
        (``shared``: what they share)."""
        new = {"starts": starts, "max_new": max_new}
        those = {"seqs": seqs} if shared is None else {"shared": shared}

        def attend(layer, q, k, v):
            q = cache.append(k, v, layer=layer, rotary=self.rotary, q=q, seqs=seqs, **new)
            return cache.attend(q, layer=layer, **those, **new, **self.seen(layer))

        return self(tokens, attend)

    def at_once(self, tokens):
        """One whole sequence, without a cache."""
        positions = torch.arange(len(tokens), dtype=torch.int32, device=tokens.device)
        starts = torch.tensor([0, len(tokens)], dtype=torch.int32, device=tokens.device)

        def attend(layer, q, k, v):
            q, k = self.rotary.apply(q, k, positions=positions)
            return window_attention(self.ctx, q, k, v, starts=starts, **self.seen(layer))

        return self(tokens, attend)


def main(branches: int = 4, steps: int = 12, found: int = 3, dim: int = 128,
         eight_bits: bool = False, states: bool = False) -> float:
    ctx = Context(0)
    dev = torch.device("cuda", ctx.device)
    g = torch.Generator().manual_seed(1)
    documents = torch.randint(VOCABULARY, (DOCUMENTS, LENGTH), generator=g).to(dev)
    vectors = torch.randn(DOCUMENTS, dim, generator=g)
    question = torch.randint(VOCABULARY, (7,), generator=g).to(dev)

    # retrieve
    query = (vectors[123] + 0.1 * torch.randn(dim, generator=g))[None].to(dev)
    _, ids = VectorDatabase(ctx, vectors).search(query, found, "cosine")
    print("documents", ids[0].tolist())
    prompt = torch.cat([documents[ids[0]].flatten(), question])

    # the prompt into the cache, slot 0
    model = Decoder(ctx, eight_bits=eight_bits)
    if states:
        model.look_at(model.embedding[documents[ids[0]]])
    longest = len(prompt) + steps
    cache = PagedKVCache(ctx, pages=(branches + 2) * (longest // 16 + 2), page_size=16,
                         kv_heads=model.kv_heads, head_dim=model.head_dim, slots=branches + 1,
                         width=longest // 16 + 1, layers=model.layers, dtype=model.dtype)
    cache.reserve([0], [len(prompt)])
    logits = model.over_cache(prompt, cache, [0], starts=[0, len(prompt)], max_new=len(prompt))

    # branches of it: whole pages are shared, each starts with another token
    slots = torch.arange(1, branches + 1, dtype=torch.int32, device=dev)
    cache.fork(torch.zeros_like(slots), slots)
    ones = torch.ones_like(slots)
    shared = cache.share([0, branches], seqs=slots)
    texts = [logits[-1].topk(branches).indices]
    for _ in range(steps):
        cache.reserve(slots, ones)
        logits = model.over_cache(texts[-1], cache, slots, shared=shared)
        texts.append(logits.argmax(1))
    assert cache.missing() == 0
    for b, text in enumerate(torch.stack(texts[:-1], 1).tolist()):
        print("branch", b, text)

    # the last step's logits against the whole sequences
    worst = 0.0
    for b in range(branches):
        whole = torch.cat([prompt, torch.stack(texts[:-1], 1)[b]])
        worst = max(worst, float((model.at_once(whole)[-1] - logits[b]).abs().max()
                                 / logits[b].abs().max()))

    held = int((cache.refs > 0).sum())
    cache.free(slots[1:])
    used = int(cache.compact())
    print("pages", held, "with every branch,", used, "with one")
    last = model.embedding.new_zeros(1, model.heads, model.head_dim) + 1
    assert bool(torch.isfinite(cache.attend(last, seqs=[1])).all())
    print(f"largest difference to the sequences at once: {worst:.4f} of the largest logit")
    return worst


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--branches", type=int, default=4)
    p.add_argument("--steps", type=int, default=12)
    p.add_argument("--eight-bits", action="store_true", help="8-bit projections")
    p.add_argument("--states", action="store_true", help="cross attention to the documents")
    a = p.parse_args()
    main(a.branches, a.steps, eight_bits=a.eight_bits, states=a.states)
