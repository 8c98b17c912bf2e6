"""Cross attention and shared prefixes in 32 bits by row tiles of 128 where scores
are large: past 2^32 times the scale, where their products with the scale are
rounded by more than a weight's range.

Each query and key has one number that is not zero, a power of two and a small
whole number, so the scores are exact, and two scores that differ do so by more
than 2^29: every key but those of a row's largest score has the weight 0, these
the weight 1.  Of n such keys the output is off by n + 2 roundings of 2^-24 of
the largest value (n - 1 sums, the division, the product, the output).  The
logarithm of the sum has seven roundings of 2^-24 of the scaled score: the
scale, log2(e), their product, the score's, the sum with log2(n), ln(2) and its
product."""
import pytest
import torch

from test_gpu_kvcache import kernels_of
from test_gpu_shared import F32, cache_of, gen, ints, keys_of, normal, starts_of

pytestmark = pytest.mark.gpu


def large(g, count, heads, d, step, low, high):
    """count x heads x d, each row step times a whole number of low to high in
    its first place."""
    x = torch.zeros(count, heads, d)
    x[..., 0] = step * torch.randint(low, high + 1, (count, heads), generator=g).float()
    return x.to("cuda:0")


def check_rows(out, lse, q, k, v, pos, scale):
    out, lse, q, k, v = (x.cpu().double() for x in (out, lse, q, k, v))
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        s = q[:, h] @ k[:, h // group].T
        s.masked_fill_(torch.arange(len(k)) > torch.as_tensor(pos)[:, None], -torch.inf)
        top = s.amax(1, keepdim=True)
        assert bool((top.abs() >= 2.0 ** 32).all())
        w = (s == top).double()
        n = w.sum(1, keepdim=True)
        want = w @ v[:, h // group] / n
        tol = 2.0 ** -24 * (n + 2) * v.abs().max()
        assert bool(((out[:, h] - want).abs() <= tol).all())
        sums = top * scale + n.log()
        assert bool(((lse[:, h] - sums[:, 0]).abs() <= 7 * 2.0 ** -24 * sums[:, 0].abs()).all())


@pytest.mark.parametrize("d", [80, 128])
@pytest.mark.parametrize("sign", [1, -1])
def test_cross(ctx, d, sign):
    """Whole sets and sets in parts, scores of one sign and of both."""
    from vectorstorekit_amd import cross_attention

    g = gen(d)
    new = [300, 5, 0, 129, 64] + [3] * 120
    keys = [1100, 33, 40, 700, 1] + [2] * 120
    at, ks = starts_of(new), starts_of(keys)
    q = large(g, at[-1], 8, d, 2.0 ** 20, 1, 3) * sign
    k = large(g, ks[-1], 2, d, 2.0 ** 13, 1, 30)
    if sign > 0:
        k[::3] *= -1
    v = normal(g, ks[-1], 2, d)
    (out, lse), used = kernels_of(ctx, lambda: cross_attention(
        ctx, q, k, v, starts=at, k_starts=ks, max_length=300, max_keys=1100,
        return_lse=True))
    assert "attn_tile32" in used
    for i in range(len(new)):
        a, b = slice(at[i], at[i + 1]), slice(ks[i], ks[i + 1])
        check_rows(out[a], lse[a], q[a], k[b], v[b], [keys[i]] * new[i], d ** -0.5)


@pytest.mark.parametrize("d", [80, 128])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("known", [True, False])
def test_shared(ctx, d, sign, known):
    """Prefixes by tiles of 128, own keys by those or, where a bound says that
    they are few, by tiles of 16."""
    from vectorstorekit_amd import PagedKVCache

    g = gen(d)
    new = [100, 7, 130, 64, 90, 1, 33, 128]
    small, slots = cache_of(ctx, g, [(2000, [150, 20, 140, 70]), (96, [100, 3, 50, 131])], 16, 2,
                            d, F32)
    small.k.copy_(large(g, small.k.shape[0] * 16, 2, d, 2.0 ** 13, 1, 30).view_as(small.k))
    table = torch.full((small.slots, 1100), -1, dtype=torch.int32, device="cuda:0")
    table[:, :small.width] = small.table
    cache = PagedKVCache.over(ctx, small.k, small.v, table, small.lengths)
    at = starts_of(new)
    q = large(g, at[-1], 8, d, 2.0 ** 20, 1, 3) * sign
    plan = cache.share(ints([0, 4] + [8] * 8), members=4, prefix=17400 if known else None)
    assert plan.prefix.tolist() == [2000] * 4 + [96] * 4 + [0]
    (out, lse), used = kernels_of(ctx, lambda: cache.attend(
        q, shared=plan, starts=at, max_new=130, return_lse=True))
    assert "attn_tile32" in used and ("attn_forms" in used) == known
    for i, slot in enumerate(slots):
        a, (k, v) = slice(at[i], at[i + 1]), keys_of(cache, slot)
        pos = range(len(k) - new[i], len(k))
        check_rows(out[a], lse[a], q[a], k, v, pos, d ** -0.5)
