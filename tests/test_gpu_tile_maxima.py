"""Row tiles of 128: the largest score of a row is that of finished products.

Calls give the same bits every time, and scores whose last places make them grow
from key to key by more than a tile's weights may grow (a maximum taken from sums
that lack their last products is too small by hundreds, and an f16 weight then
infinite) come out as the definition has them.  Tolerances: test_gpu_shared.py."""
import pytest
import torch

from test_gpu_kvcache import kernels_of
from test_gpu_shared import (BF, F16, F32, attended, cache_of, check, check_lse, check_shared, gen,
                             normal, starts_of)

pytestmark = pytest.mark.gpu

#: heads, key heads, dimension
HEADS = [(8, 2, 64), (12, 3, 96), (16, 4, 128), (16, 2, 256)]
TILE = {BF: "attn_tile", F16: "attn_tile", F32: "attn_tile32"}


def growing(g, count, heads, d, dtype, least, most):
    """count x heads x d: nothing but in the last 16 places, which grow from row
    to row from `least` to `most`, and a little noise in them."""
    x = torch.zeros(count, heads, d)
    ramp = torch.linspace(least, most, count)[:, None, None]
    x[..., -16:] = ramp + 0.01 * torch.randn(count, heads, 16, generator=g)
    return x.to(dtype).to("cuda:0")


def prompt(ctx, g, dtype, heads, kv, d, make):
    """Causal, over keys of their own."""
    from vectorstorekit_amd import window_attention

    new = [700, 129, 64, 1, 300]
    at = starts_of(new)
    q, k = make(at[-1], heads, True), make(at[-1], kv, False)
    v = normal(g, at[-1], kv, d, dtype=dtype)

    def checked(out, lse):
        for i, t in enumerate(new):
            a = slice(at[i], at[i + 1])
            want, sums, tol = attended(q[a], k[a], v[a], range(t), d ** -0.5)
            check(out[a], want, tol)
            check_lse(lse[a], sums)
    return lambda: window_attention(ctx, q, k, v, starts=at, max_length=700,
                                    return_lse=True), checked


def cross(ctx, g, dtype, heads, kv, d, make):
    from vectorstorekit_amd import cross_attention

    new, keys = [400, 129, 64, 1, 300] + [2] * 60, [1500, 300, 65, 700, 64] + [3] * 60
    at, ks = starts_of(new), starts_of(keys)
    q, k = make(at[-1], heads, True), make(ks[-1], kv, False)
    v = normal(g, ks[-1], kv, d, dtype=dtype)

    def checked(out, lse):
        for i, t in enumerate(new):
            a, b = slice(at[i], at[i + 1]), slice(ks[i], ks[i + 1])
            want, sums, tol = attended(q[a], k[b], v[b], [keys[i]] * t, d ** -0.5)
            check(out[a], want, tol)
            check_lse(lse[a], sums)
    return lambda: cross_attention(ctx, q, k, v, starts=at, k_starts=ks, max_length=400,
                                   max_keys=1500, return_lse=True), checked


def shared(ctx, g, dtype, heads, kv, d, make):
    from vectorstorekit_amd import PagedKVCache

    new = [100, 7, 130, 64, 90, 1, 33, 128]
    small, slots = cache_of(ctx, g, [(2000, [150, 20, 140, 70]), (96, [100, 3, 50, 131])], 16, kv,
                            d, dtype)
    # (pages in no order: a page's number is its place in what grows)
    small.k.copy_(make(small.k.shape[0] * 16, kv, False).view_as(small.k))
    table = torch.full((small.slots, 1100), -1, dtype=torch.int32, device="cuda:0")
    table[:, :small.width] = small.table
    cache = PagedKVCache.over(ctx, small.k, small.v, table, small.lengths)
    at = starts_of(new)
    q = make(at[-1], heads, True)
    plan = cache.share([0, 4] + [8] * 8, members=4)
    return (lambda: cache.attend(q, shared=plan, starts=at, max_new=130, return_lse=True),
            lambda out, lse: check_shared(cache, slots, q, at, out, d ** -0.5, lse))


CASES = [(form, dtype, *h) for form in (prompt, cross, shared) for dtype in (BF, F16, F32)
         for h in HEADS if dtype != F32 or form is not prompt and 64 < h[2] <= 128]


@pytest.mark.parametrize("form,dtype,heads,kv,d", CASES)
def test_scores_that_grow(ctx, form, dtype, heads, kv, d):
    g = gen(d)
    call, checked = form(ctx, g, dtype, heads, kv, d, lambda n, h, q: growing(
        g, n, h, d, dtype, *((12.0, 16.0) if q else (0.0, 20.0))))
    (out, lse), used = kernels_of(ctx, call)
    assert TILE[dtype] in used
    checked(out, lse)


@pytest.mark.parametrize("form,dtype,heads,kv,d", CASES)
def test_the_same_bits(ctx, form, dtype, heads, kv, d):
    g = gen(d)
    call, checked = form(ctx, g, dtype, heads, kv, d,
                         lambda n, h, q: normal(g, n, h, d, dtype=dtype))
    (out, lse), used = kernels_of(ctx, call)
    assert TILE[dtype] in used
    checked(out, lse)
    for _ in range(12):
        again, sums = call()
        assert torch.equal(again, out) and torch.equal(sums, lse)
