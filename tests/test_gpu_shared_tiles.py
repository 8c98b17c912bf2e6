"""Cross attention and shared prefixes by row tiles of 128 in 16 bits, by the
names that profiling reports: prefixes beside own keys in one launch, in two,
both by tiles; parts; several sequences of one set; masked places that are not
finite; scores past what the tile's scaled sums hold.  Tolerances as in
test_gpu_shared.py, and test_gpu_large_scores.py for the last."""
import math

import pytest
import torch

from test_gpu_kvcache import kernels_of
from test_gpu_large_scores import large
from test_gpu_shared import (BF, F16, attended, cache_of, check, check_lse, check_shared, gen,
                             keys_of, normal, starts_of)

pytestmark = pytest.mark.gpu
U = {BF: 2.0 ** -8, F16: 2.0 ** -11}


def branches(ctx, heads, kv, d, dtype, sizes, new, seed=0):
    """Groups of 1,040 shared keys, of 496, of 48, a sequence alone and some that
    share nothing; as many members as said; up to `new` new tokens each, none
    among them, more than some have keys of their own; NaN behind every end.
    The cache, its slots, the groups' offsets and the tokens' offsets."""
    g = gen(d + new + seed)
    tails = [torch.randint(1, 60, (m,), generator=g).tolist() for m in sizes]
    shared = (1040, 496, 48, 320, 0)
    order = torch.randperm(sum(sizes), generator=g).tolist()
    cache, slots = cache_of(ctx, g, list(zip(shared, tails)), 16, kv, d, dtype, order=order)
    counts = torch.randint(0, new + 1, (len(slots),), generator=g).tolist()
    counts[0] = new
    counts = [min(c, int(cache.lengths[s])) for c, s in zip(counts, slots)]
    for s in slots:
        length = int(cache.lengths[s])
        if length % 16:
            page = int(cache.table[s, length // 16])
            cache.k[page, length % 16:], cache.v[page, length % 16:] = math.nan, math.inf
    return cache, slots, starts_of(sizes), starts_of(counts), normal(
        g, sum(counts), heads, d, dtype=dtype)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("heads,kv,d,sizes,new,kernels", [
    (32, 4, 64, (64, 7, 2, 1, 3), 3, {"attn_shared"}),
    (16, 4, 80, (64, 7, 2, 1, 3), 4, {"attn_shared"}),
    (32, 4, 96, (40, 9, 5, 1, 2), 3, {"attn_shared"}),
    (16, 4, 128, (70, 7, 2, 1, 3), 4, {"attn_shared"}),
    (28, 4, 128, (33, 16, 3, 1, 2), 3, {"attn_shared"}),
    # a head that leaves no room for both in one launch
    (16, 2, 256, (64, 7, 2, 1, 3), 4, {"attn_tile", "attn_forms"}),
    (8, 1, 200, (90, 30, 20, 1, 9), 6, {"attn_tile", "attn_forms"}),
    # own keys by tiles too, in one launch
    (32, 4, 64, (25, 5, 3, 1, 3), 20, {"attn_tile"}),
    (16, 4, 128, (30, 5, 3, 1, 4), 20, {"attn_tile"}),
    (24, 3, 72, (25, 5, 3, 1, 3), 20, {"attn_tile"}),
    (16, 2, 256, (25, 5, 3, 1, 3), 20, {"attn_tile"})])
@pytest.mark.parametrize("known", [False, True])
def test_shared(ctx, dtype, heads, kv, d, sizes, new, kernels, known):
    cache, slots, offsets, at, q = branches(ctx, heads, kv, d, dtype, sizes, new)
    plan = cache.share(offsets, seqs=slots, prefix=1040 if known else None)
    n = plan.prefix.tolist()
    assert [n[i] for i in offsets[:3]] == [1040, 496, 48] and n[-1] == 0
    attend = lambda: cache.attend(q, shared=plan, starts=at, max_new=new, return_lse=True,
                                  max_length=1100 if known else None)
    (out, lse), used = kernels_of(ctx, attend)
    assert used == kernels | {"attn_join"}
    check_shared(cache, slots, q, at, out, d ** -0.5, lse)
    # members cut back: into the prefix, to its end, to their new tokens
    lengths = cache.lengths.clone()
    for i, left in ((0, 700), (1, 1040), (2, max(new, 1)), (offsets[1], 100)):
        if left >= at[i + 1] - at[i]:
            cache.lengths[slots[i]] = left
    out, lse = attend()
    check_shared(cache, slots, q, at, out, d ** -0.5, lse)
    cache.lengths.copy_(lengths)


@pytest.mark.parametrize("heads,kv,d", [(32, 4, 64), (16, 4, 128), (16, 2, 256)])
def test_shared_captured(ctx, heads, kv, d):
    """Replays over other queries, with eager work between, give what the eager
    call gives; so do two streams at once."""
    sizes, new = (64, 7, 2, 1, 3), 4
    cache, slots, offsets, at, q = branches(ctx, heads, kv, d, BF, sizes, new)
    plan = cache.share(offsets, seqs=slots)
    starts = torch.tensor(at, dtype=torch.int32, device="cuda:0")
    attend = lambda: cache.attend(q, shared=plan, starts=starts, max_new=new)
    attend()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend()
    g = gen(1)
    for _ in range(4):
        q.copy_(normal(g, *q.shape, dtype=BF))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, attend())
    check_shared(cache, slots, q, at, got, d ** -0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [attend() for _ in range(3)]
    here = [attend() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, got) for x in there + here)


# heads, key heads, their dimension; new tokens; keys of the sets; each sequence's
# set; parts are joined
CROSS = [
    (8, 2, 64, [200, 1, 0, 77, 150, 129, 33], [5000, 900, 0, 64], [0, 1, 0, 2, 3, 0, 1], True),
    (16, 4, 128, [100, 33, 0, 128, 5], [4000, 65, 0, 1000], [0, 0, 1, 3, 2], True),
    (16, 2, 256, [130, 64, 7, 90], [3000, 0, 500], [0, 2, 1, 0], True),
    (12, 4, 96, [150, 90, 3, 0, 200, 60], [2500, 1, 33], [0, 0, 2, 1, 0, 7], True),
    (32, 8, 128, [300, 129, 1, 64, 250, 90], [700, 64, 0, 63, 129, 1], None, False),
    (8, 8, 64, [700, 400, 64, 63, 1, 650], [300, 129, 1, 0, 65, 257], None, False),
    (20, 5, 80, [200, 128, 127, 0, 1, 64] * 2, [500, 1, 64, 0, 70, 255], [0, 1, 2, 3, 4, 5] * 2,
     False),
    (8, 1, 256, [300, 200, 129, 0, 9], [400, 33, 32, 1, 0], [0, 1, 2, 3, 4], False)]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("heads,kv,d,new,keys,sets,parts", CROSS)
@pytest.mark.parametrize("padded", [False, True])
def test_cross(ctx, dtype, heads, kv, d, new, keys, sets, parts, padded):
    """Behind a padded set's keys nothing finite; an infinite value that all see
    is its column's result."""
    from vectorstorekit_amd import cross_attention

    g = gen(d + sum(new))
    at, ks = starts_of(new), starts_of(keys)
    q = normal(g, at[-1], heads, d, dtype=dtype)
    k, v = (normal(g, ks[-1], kv, d, dtype=dtype) for _ in range(2))
    if padded:
        pk, pv = (torch.full((len(keys), max(keys), kv, d), x, dtype=dtype, device="cuda:0")
                  for x in (math.nan, -math.inf))
        for i, n in enumerate(keys):
            pk[i, :n], pv[i, :n] = k[ks[i]:ks[i + 1]], v[ks[i]:ks[i + 1]]
        call = lambda: cross_attention(ctx, q, pk, pv, starts=at, k_lengths=keys, sets=sets,
                                       max_length=max(new), return_lse=True)
    else:
        call = lambda: cross_attention(ctx, q, k, v, starts=at, k_starts=ks, sets=sets,
                                       max_length=max(new), max_keys=max(keys), return_lse=True)
    (out, lse), used = kernels_of(ctx, call)
    assert used == ({"attn_tile", "attn_join"} if parts else {"attn_tile"})
    which = sets or range(len(new))

    def checked(out, lse, v):
        for i, z in enumerate(which):
            a = slice(at[i], at[i + 1])
            b = slice(ks[z], ks[z + 1]) if z < len(keys) else slice(0, 0)
            want, sums, tol = attended(q[a], k[b], v[b], [10 ** 6] * new[i], d ** -0.5)
            check(out[a], want, tol)
            check_lse(lse[a], sums)

    checked(out, lse, v)
    # in the middle of the longest set, and its last value
    clean = v.clone()
    for j, e, x in ((keys[0] // 2, 3, math.inf), (keys[0] - 1, d - 1, -math.inf)):
        v[j, 0, e], clean[j, 0, e] = x, 0.0
        if padded:
            pv[0, j, 0, e] = x
    out, lse = call()
    for i, z in enumerate(which):
        if z == 0:
            rows = out[at[i]:at[i + 1], :heads // kv]
            assert bool((rows[..., 3] == math.inf).all())
            assert bool((rows[..., d - 1] == -math.inf).all())
    finite = out.clone()
    bare, _ = cross_attention(ctx, q, k, clean, starts=at, k_starts=ks, sets=sets,
                              max_length=max(new), max_keys=max(keys), return_lse=True)
    hot = torch.isinf(out)
    finite[hot] = bare[hot]
    checked(finite, lse, clean)


def check_tops(dtype, out, lse, q, k, v, pos, scale):
    """Rows whose weights are 1 for the largest score's keys and 0 for the others
    (test_gpu_large_scores.py), here each rounded once with the output: two
    roundings of the type more."""
    out, lse, q, k, v = (x.cpu().double() for x in (out, lse, q, k, v))
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        s = q[:, h] @ k[:, h // group].T
        s.masked_fill_(torch.arange(len(k)) > torch.as_tensor(pos)[:, None], -torch.inf)
        top = s.amax(1, keepdim=True)
        w = (s == top).double()
        n = w.sum(1, keepdim=True)
        tol = (2 * U[dtype] + 2.0 ** -24 * (n + 2)) * v.abs().max()
        assert bool(((out[:, h] - w @ v[:, h // group] / n).abs() <= tol).all())
        sums = top * scale + n.log()
        assert bool(((lse[:, h] - sums[:, 0]).abs() <= 7 * 2.0 ** -24 * sums[:, 0].abs()).all())


STEPS = {BF: (2.0 ** 20, 2.0 ** 13), F16: (2.0 ** 14, 2.0 ** 10)}


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("heads,kv,d,new,keys,parts", [
    (16, 4, 64, [200, 1, 130], [5000, 900, 64], True),
    (16, 4, 128, [100, 33, 128], [4000, 65, 1000], True),
    (32, 8, 128, [300, 129, 1, 64, 250, 90], [700, 64, 9, 63, 129, 1], False),
    (16, 2, 256, [130, 64, 7, 90], [3000, 5, 500, 70], True)])
def test_cross_large_scores(ctx, dtype, sign, heads, kv, d, new, keys, parts):
    from vectorstorekit_amd import cross_attention

    g = gen(d)
    a, b = STEPS[dtype]
    at, ks = starts_of(new), starts_of(keys)
    q = (large(g, at[-1], heads, d, a, 1, 3) * sign).to(dtype)
    k = large(g, ks[-1], kv, d, b, 1, 30)
    if sign > 0:
        k[::3] *= -1
    k, v = k.to(dtype), normal(g, ks[-1], kv, d, dtype=dtype)
    (out, lse), used = kernels_of(ctx, lambda: cross_attention(
        ctx, q, k, v, starts=at, k_starts=ks, max_length=max(new), max_keys=max(keys),
        return_lse=True))
    assert used == ({"attn_tile", "attn_join"} if parts else {"attn_tile"})
    for i in range(len(new)):
        x, y = slice(at[i], at[i + 1]), slice(ks[i], ks[i + 1])
        check_tops(dtype, out[x], lse[x], q[x], k[y], v[y], [keys[i]] * new[i], d ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("heads,kv,d,sizes,new,kernels", [
    (32, 4, 64, (64, 7, 2, 1, 3), 3, {"attn_shared"}),
    (16, 4, 128, (70, 7, 2, 1, 3), 4, {"attn_shared"}),
    (16, 2, 256, (64, 7, 2, 1, 3), 4, {"attn_tile", "attn_forms"}),
    (16, 4, 128, (30, 5, 3, 1, 4), 20, {"attn_tile"})])
def test_shared_large_scores(ctx, dtype, sign, heads, kv, d, sizes, new, kernels):
    cache, slots, offsets, at, q = branches(ctx, heads, kv, d, dtype, sizes, new)
    g = gen(d)
    a, b = STEPS[dtype]
    q.copy_(large(g, len(q), heads, d, a, 1, 3) * sign)
    cache.k.copy_(large(g, cache.k.shape[0] * 16, kv, d, b, 1, 30).view_as(cache.k))
    cache.v.copy_(normal(g, *cache.v.shape, dtype=dtype))
    plan = cache.share(offsets, seqs=slots)
    (out, lse), used = kernels_of(ctx, lambda: cache.attend(
        q, shared=plan, starts=at, max_new=new, return_lse=True))
    assert used == kernels | {"attn_join"}
    for i, slot in enumerate(slots):
        t = at[i + 1] - at[i]
        if t:
            x, (k, v) = slice(at[i], at[i + 1]), keys_of(cache, slot)
            check_tops(dtype, out[x], lse[x], q[x], k, v, range(len(k) - t, len(k)), d ** -0.5)
