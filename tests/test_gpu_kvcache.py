"""Key-value cache, rotary positions and attention against their definitions
in 64 bits.

Tolerances, derived here and used by every case.  With u the unit roundoff of
the output's type (2^-8 bf16, 2^-11 f16, 2^-24 f32):

* a rotated value: one rounding u of the result, fp32 products and a sine and
  cosine that are off by at most 2^-18 (16-bit types) or 2^-22: |err| <=
  u |y| + 2^-17 (|a| + |b|) A, or + 2^-21 (...) for f32;
* an attention output: the score of fp32 products is off by at most
  e = 2^-24 (d + 8) scale max sum |q k|, a weight by a factor within
  e + 2^-21, the sum of L weights by 2^-24 (L + 16); 16-bit types may round
  each weight once (u); so |err| <= u |o| + max |v| (2 (e + 2^-21 +
  2^-24 (L + 16)) + (16-bit) u), and the errors are independent, so their
  2-norm is at most u (16-bit) of the result's."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda:0"


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, dtype=torch.float32).to(dtype).to(DEV)


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ definitions

def rotated(x, positions, inv, amplitude, layout, sign=1.0):
    """x (tokens x heads x d) turned, in 64 bits on the CPU."""
    y = x.detach().cpu().double().clone()
    r = 2 * len(inv)
    angle = positions.cpu().double()[:, None] * torch.from_numpy(inv)
    c, s = torch.cos(angle)[:, None] * amplitude, sign * torch.sin(angle)[:, None] * amplitude
    i = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    a, b = y[..., i[0]].clone(), y[..., i[1]].clone()
    y[..., i[0]], y[..., i[1]] = a * c - b * s, a * s + b * c
    return y


def attended(q, k, v, scale, window, sinks):
    """One sequence: q (T x H x d) the last tokens of k, v (L x Hkv x d), in 64
    bits on the CPU.  Only what a row sees enters its sums.  Returns the
    outputs, the logarithms of the sums, and the tolerance of each output."""
    t, heads, d = q.shape
    dtype = q.dtype
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    length, kv = k.shape[0], k.shape[1]
    out = torch.zeros(t, heads, d, dtype=torch.float64)
    lse = torch.full((t, heads), -math.inf, dtype=torch.float64)
    tol = torch.zeros(t, heads, d, dtype=torch.float64)
    j = torch.arange(length)
    u = U[dtype]
    for i in range(t):
        pos = length - t + i
        see = j <= pos
        if window:
            see &= (pos - j < window) | (j < sinks)
        if not see.any():
            continue
        for h in range(heads):
            kk, vv = k[see, h // (heads // kv)], v[see, h // (heads // kv)]
            s = kk @ q[i, h] * scale
            lse[i, h] = torch.logsumexp(s, 0)
            out[i, h] = torch.softmax(s, 0) @ vv
            e = 2.0 ** -24 * (d + 8) * scale * float((kk.abs() @ q[i, h].abs()).max())
            w = 2 * (e + 2.0 ** -21 + 2.0 ** -24 * (length + 16)) + (u if u > 2.0 ** -20 else 0)
            tol[i, h] = u * out[i, h].abs() + float(vv.abs().max()) * w
    return out, lse, tol


def check(got, want, tol):
    got = got.detach().cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    err = (got - want).abs()[fine]
    assert bool((err <= tol[fine]).all()), float((err - tol[fine]).max())


def check_norm(got, want, dtype):
    if dtype != F32 and float(want.norm()) > 0:
        assert float((got.cpu().double() - want).norm()) <= U[dtype] * float(want.norm())


# ------------------------------------------------------------------------ rotary

@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r,tokens,heads,kv", [(128, 128, 7, 8, 2), (80, 32, 33, 5, 5),
                                                 (96, 48, 1, 3, 1), (64, 40, 300, 2, 1),
                                                 (37, 10, 5, 3, 3), (256, 256, 2, 1, 1),
                                                 (2, 2, 9, 1, 1)])
def test_rotary(ctx, dtype, layout, d, r, tokens, heads, kv):
    from vectorstorekit_amd import RotaryEmbedding

    g = gen(d + r)
    rope = RotaryEmbedding(ctx, d, rotary_dim=r, layout=layout)
    q, k = normal(g, tokens, heads, d, dtype=dtype), normal(g, tokens, kv, d, dtype=dtype)
    pos = torch.randint(-5000, 1 << 20, (tokens,), generator=g, dtype=torch.int32).to(DEV)
    pos[0] = 2 ** 31 - 1
    for inverse in (False, True):
        for x, y in zip((q, k), rope.apply(q, k, positions=pos, inverse=inverse)):
            want = rotated(x, pos, rope.inv_freq, 1.0, layout, -1.0 if inverse else 1.0)
            size = x.cpu().double().abs().amax(-1, keepdim=True)
            e = 2.0 ** -21 if dtype == F32 else 2.0 ** -17
            check(y, want, U[dtype] * want.abs() + 2 * e * size)
            assert torch.equal(y[..., r:], x[..., r:])
    back = rope.apply(q, positions=pos)
    assert torch.equal(back, rope.apply(q, k, positions=pos)[0])
    z = q.clone()
    assert rope.apply(z, positions=pos, inplace=True) is z and torch.equal(z, back)
    rope.free()


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 4.0},
                                     {"type": "ntk", "factor": 8.0},
                                     {"type": "yarn", "factor": 8.0, "original_length": 4096},
                                     {"type": "yarn", "factor": 2.0, "original_length": 512,
                                      "beta_fast": 16, "beta_slow": 2, "attention_factor": 1.5}])
def test_rotary_scaled(ctx, scaling):
    from vectorstorekit_amd import RotaryEmbedding

    rope = RotaryEmbedding(ctx, 64, scaling=scaling, base=5000.0)
    inv = np.array([5000.0 ** (-2 * i / 64) for i in range(32)])
    amplitude, f = 1.0, scaling["factor"]
    if scaling["type"] == "linear":
        inv = inv / f
    elif scaling["type"] == "ntk":
        # the slowest pair is divided by f, the fastest stays
        ntk = [5000.0 ** (-2 * i / 64) * f ** (-2 * i / 62) for i in range(32)]
        inv = np.array(ntk)
        assert abs(inv[-1] * f / 5000.0 ** (-62 / 64) - 1) < 1e-12 and inv[0] == 1
    else:
        n, fast, slow = scaling["original_length"], scaling.get("beta_fast", 32), scaling.get("beta_slow", 1)
        turns = n * inv / (2 * math.pi)
        at = [64 * math.log(n / (2 * math.pi * b)) / (2 * math.log(5000.0)) for b in (fast, slow)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), 63)
        ramp = np.clip((np.arange(32) - low) / (high - low), 0, 1)
        assert np.all(ramp[turns > fast * 1.5] == 0) and np.all(ramp[turns < slow / 1.5] == 1)
        inv = inv * (1 - ramp) + inv / f * ramp
        amplitude = scaling.get("attention_factor", 0.1 * math.log(f) + 1)
    np.testing.assert_allclose(rope.inv_freq, inv, rtol=1e-12)
    x = normal(gen(1), 50, 2, 64)
    pos = ints(range(0, 50 * 997, 997))
    want = rotated(x, pos, inv, amplitude, "half")
    check(rope.apply(x, positions=pos), want, 2.0 ** -24 * want.abs()
          + 2.0 ** -20 * x.cpu().double().abs().amax(-1, keepdim=True) * amplitude)


def test_rotary_strides_and_gradient(ctx):
    """Sliced inputs, and the inverse as the gradient: <R x, y> = <x, R' y>,
    the formula's, and the differences of the (linear) forward."""
    from vectorstorekit_amd import RotaryEmbedding

    g = gen(2)
    rope = RotaryEmbedding(ctx, 48, rotary_dim=32, layout="interleaved",
                           scaling={"type": "yarn", "factor": 4.0, "original_length": 1024})
    packed = normal(g, 21, 3, 6, 48)  # q, k, v of one projection
    q, k = packed[:, 0], packed[:, 1, :2]
    pos = ints(range(40, 61))
    a, b = rope.apply(q, k, positions=pos)
    assert torch.equal(a, rope.apply(q.contiguous(), positions=pos))
    assert torch.equal(b, rope.apply(k.contiguous(), positions=pos))
    t = q.transpose(1, 2).contiguous().transpose(1, 2)  # heads not dense
    assert torch.equal(a, rope.apply(t, positions=pos))
    y = normal(g, 21, 6, 48)
    grad = rope.apply(y, positions=pos, inverse=True)
    want = rotated(y, pos, rope.inv_freq, rope.amplitude, "interleaved", -1.0)
    check(grad, want, 2.0 ** -24 * want.abs()
          + 2.0 ** -20 * y.cpu().double().abs().amax(-1, keepdim=True) * rope.amplitude)
    e = normal(g, 21, 6, 48)
    h = 0.5
    up, down = (rope.apply((q + f * e).contiguous(), positions=pos) for f in (h, -h))
    slope = float(((up - down).double() * y.double()).sum()) / (2 * h)
    # the sums of 21 * 6 * 48 products, each off by 2^-20 of its size
    size = float((e.double().abs() * y.double().abs()).sum()) * 4
    assert abs(slope - float((e.double() * grad.double()).sum())) <= 2.0 ** -20 * size


def test_given_frequencies(ctx):
    """Frequencies of the caller's own, zeros and fast ones among them."""
    from vectorstorekit_amd import RotaryEmbedding, VSKError

    inv = np.concatenate([[0.0, 3.0, 1e-7], 7.0 ** -np.arange(17)])
    x, pos = normal(gen(6), 40, 3, 64), ints(range(0, 40 * 5003, 5003))
    for scaling, a in (({"type": "given", "inv_freq": inv}, 1.0),
                       ({"type": "given", "inv_freq": inv.tolist(), "attention_factor": 1.25}, 1.25)):
        rope = RotaryEmbedding(ctx, 64, rotary_dim=40, scaling=scaling)
        assert rope.amplitude == a and rope.inv_freq.tolist() == inv.tolist()
        want = rotated(x, pos, inv, a, "half")
        check(rope.apply(x, positions=pos), want, 2.0 ** -24 * want.abs()
              + 2.0 ** -20 * x.cpu().double().abs().amax(-1, keepdim=True) * a)
    for bad in ({"type": "given"}, {"type": "given", "inv_freq": inv[:3]},
                {"type": "given", "inv_freq": inv, "factor": 2.0},
                {"type": "given", "inv_freq": -inv}, {"type": "given", "inv_freq": inv + math.inf}):
        with pytest.raises(VSKError) as e:
            RotaryEmbedding(ctx, 64, rotary_dim=40, scaling=bad)
        assert e.value.kind == "invalidArgument"


@pytest.mark.parametrize("scaling", [None, {"type": "yarn", "factor": 8.0,
                                            "original_length": 512}])
def test_moved_keys(ctx, scaling):
    """A turned key moved to another position, by the inverse, is that key
    turned there, times the factor.  Three rotations, each off by 2^-24 of the
    value and 2^-21 of the pair's size."""
    from vectorstorekit_amd import RotaryEmbedding

    rope = RotaryEmbedding(ctx, 64, scaling=scaling)
    a = rope.amplitude
    assert (a == 1.0) == (scaling is None)
    x, p, to = normal(gen(4), 30, 2, 64), ints(range(1000, 1030)), ints(range(30))
    moved = rope.apply(rope.apply(x, positions=p), positions=p - to, inverse=True)
    want = rope.apply(x, positions=to).cpu().double() * a
    size = x.cpu().double().abs().amax(-1, keepdim=True) * a * a
    check(moved, want, 3 * (2.0 ** -24 * want.abs() + 2.0 ** -20 * size))


# ---------------------------------------------------------------------- the cache

def filled(ctx, lengths, page, kv, d, dtype, *, layers=1, order="nhd", seed=0, width=None,
           poison=True):
    """A cache whose sequences hold pages from all over the pool; what no
    sequence holds (page tails, free pages) is NaN.  Also each sequence's keys
    and values, layers x L x kv x d."""
    from vectorstorekit_amd import PagedKVCache

    g = gen(seed)
    used = [-(-x // page) for x in lengths]
    pages = sum(used) + 3
    width = width or max(max(used), 1)
    ids = torch.randperm(pages, generator=g).tolist()
    shape = (layers, pages, page, kv, d)
    k, v = (torch.full(shape, math.nan if poison else 0.0, dtype=dtype) for _ in range(2))
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    seqs, at = [], 0
    for s, x in enumerate(lengths):
        kk, vv = (torch.randn(layers, x, kv, d, generator=g).to(dtype) for _ in range(2))
        for i in range(used[s]):
            p = ids[at]
            at += 1
            table[s, i] = p
            n = min(page, x - i * page)
            k[:, p, :n], v[:, p, :n] = kk[:, i * page:i * page + n], vv[:, i * page:i * page + n]
        seqs.append((kk, vv))
    k, v = k.to(DEV), v.to(DEV)
    if order == "hnd":  # heads outside the page's rows
        k, v = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in (k, v))
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[table[table >= 0].long()] = 1
    cache = PagedKVCache.over(ctx, k, v, table.to(DEV), ints(lengths), refs.to(DEV))
    return cache, seqs


TOKEN = [
    # lengths, page, heads, kv, d, window, sinks
    ([1], 16, 8, 8, 64, None, 0),
    ([0, 1, 15, 16, 17, 33], 16, 8, 2, 128, None, 0),
    ([777], 16, 32, 8, 128, None, 0),
    ([2050, 3, 0, 129], 64, 4, 1, 128, 100, 4),
    ([1500], 32, 12, 12, 96, 64, 0),
    ([300, 299], 128, 20, 5, 80, 1, 1),
    ([5000, 31], 16, 9, 3, 64, 333, 40),
    ([260], 32, 8, 1, 256, None, 0),
    ([200], 16, 34, 2, 128, 50, 2),   # 17 heads a group: two row tiles
    ([90, 64], 16, 3, 1, 36, 20, 3),  # heads that take no 16-byte loads in 16 bits
    ([70], 16, 2, 2, 1, None, 0),
    ([65], 16, 2, 1, 255, 9, 0),
]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("lengths,page,heads,kv,d,window,sinks", TOKEN)
def test_token_attention(ctx, dtype, lengths, page, heads, kv, d, window, sinks):
    cache, seqs = filled(ctx, lengths, page, kv, d, dtype, layers=2, seed=d + heads)
    q = normal(gen(5), len(lengths), heads, d, dtype=dtype)
    scale = d ** -0.5
    for layer in (0, 1):
        out, lse = cache.attend(q, layer=layer, window=window, sinks=sinks, return_lse=True)
        want = [attended(q[i:i + 1], kk[layer], vv[layer], scale, window, sinks)
                for i, (kk, vv) in enumerate(seqs)]
        o, l, t = (torch.cat(x) for x in zip(*want))
        check(out, o, t)
        check_norm(out, o, dtype)
        check(lse, l, 2.0 ** -16 * (1 + l.abs()))
    # a bound of the lengths only divides the work, wrong ones included
    for bound in (1, 200, 10 ** 6):
        again = cache.attend(q, layer=1, window=window, sinks=sinks, max_length=bound)
        check(again, o, t)


def test_token_long_split(ctx):
    """A length that many parts share, and slots out of order."""
    cache, seqs = filled(ctx, [40, 70001, 5], 64, 2, 128, BF, seed=3)
    q = normal(gen(6), 2, 8, 128, dtype=BF)
    out, lse = cache.attend(q, seqs=[1, 0], scale=0.2, return_lse=True)
    for i, s in enumerate((1, 0)):
        o, l, t = attended(q[i:i + 1], seqs[s][0][0], seqs[s][1][0], 0.2, None, 0)
        check(out[i:i + 1], o, t)
        check(lse[i:i + 1], l, 2.0 ** -16 * (1 + l.abs()))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("order", ["nhd", "hnd"])
@pytest.mark.parametrize("news,lengths,page,heads,kv,d,window,sinks", [
    ([3, 1, 0, 17], [3, 90, 12, 40], 16, 4, 2, 64, None, 0),
    ([70, 130], [200, 130], 32, 8, 2, 128, 33, 4),
    ([5], [900], 64, 16, 2, 128, 200, 7),
    ([300], [300], 64, 2, 1, 96, 64, 0),
    ([65, 64, 63], [65, 100, 63], 16, 6, 6, 80, 16, 16),
    ([40, 9], [64, 20], 16, 4, 1, 256, None, 0),
    ([33], [50], 16, 3, 3, 20, 11, 1),
])
def test_prompt_attention(ctx, dtype, order, news, lengths, page, heads, kv, d, window, sinks):
    """Several new tokens a sequence over the cache, ragged."""
    cache, seqs = filled(ctx, lengths, page, kv, d, dtype, order=order, seed=d + 1)
    starts = [0] + list(np.cumsum(news))
    q = normal(gen(7), starts[-1], heads, d, dtype=dtype)
    out, lse = cache.attend(q, starts=starts, max_new=max(news), window=window, sinks=sinks,
                            return_lse=True)
    for i, (kk, vv) in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        o, l, t = attended(q[a:b], kk[0], vv[0], d ** -0.5, window, sinks)
        check(out[a:b], o, t)
        check_norm(out[a:b], o, dtype)
        check(lse[a:b], l, 2.0 ** -16 * (1 + l.abs()))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("lengths,heads,kv,d,window,sinks", [
    ([1], 2, 2, 64, 1, 0),
    ([333], 4, 4, 64, 128, 4),
    ([0, 257, 64, 1], 8, 2, 128, 100, 4),
    ([520, 31], 3, 1, 96, 64, 130),
    ([190], 4, 1, 256, 32, 0),
    ([130], 2, 2, 128, None, 0),
    ([75, 20], 5, 5, 40, 30, 2),
    ([66], 2, 1, 33, 12, 5),
])
def test_window_attention(ctx, dtype, lengths, heads, kv, d, window, sinks):
    from vectorstorekit_amd import window_attention

    g = gen(d)
    starts = [0] + list(np.cumsum(lengths))
    packed = normal(g, starts[-1], heads + 2 * kv, d, dtype=dtype)  # one projection's output
    q, k, v = packed[:, :heads], packed[:, heads:heads + kv], packed[:, heads + kv:]
    out, lse = window_attention(ctx, q, k, v, starts=starts, max_length=max(lengths),
                                window=window, sinks=sinks, return_lse=True)
    dense = window_attention(ctx, q.contiguous(), k.contiguous(), v.contiguous(),
                             starts=ints(starts), window=window, sinks=sinks)
    for i in range(len(lengths)):
        a, b = starts[i], starts[i + 1]
        o, l, t = attended(q[a:b], k[a:b], v[a:b], d ** -0.5, window, sinks)
        check(out[a:b], o, t)
        check(dense[a:b], o, t)
        check_norm(out[a:b], o, dtype)
        check(lse[a:b], l, 2.0 ** -16 * (1 + l.abs()))


def test_queries_before_the_keys(ctx):
    """More queries than keys: the first ones stand before every key, see
    nothing and get zeros."""
    from vectorstorekit_amd import window_attention

    g = gen(8)
    q, k, v = (normal(g, n, 2, 64, dtype=BF) for n in (40, 25, 25))
    out, lse = window_attention(ctx, q, k, v, starts=[0, 30, 40], k_starts=[0, 25, 25],
                                return_lse=True)
    assert not out[:5].any() and not out[30:].any()
    assert bool(torch.isneginf(lse[:5]).all()) and bool(torch.isneginf(lse[30:]).all())
    o, _, t = attended(q[5:30], k, v, 64 ** -0.5, None, 0)
    check(out[5:30], o, t)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,kv,d,n", [(4, 2, 128, 150), (2, 2, 64, 400), (4, 1, 256, 70)])
def test_masked_places_do_not_reach_sums(ctx, dtype, bad, heads, kv, d, n):
    """A key or value that is not finite reaches the rows that see it and no
    others: the masked product 0 * NaN is not taken."""
    from vectorstorekit_amd import window_attention

    g = gen(9)
    q, k, v = (normal(g, n, h, d, dtype=dtype) for h in (heads, kv, kv))
    at, window, sinks = n - 45, 20, 3
    for x, j in ((k, at), (v, at), (v, 1)):
        y = [t.clone() for t in (k, v)]
        (y[0] if x is k else y[1])[j, 0, d // 2] = bad
        out = window_attention(ctx, q, *y, starts=[0, n], window=window, sinks=sinks)
        rows = torch.arange(n)
        see = (rows >= j) & ((rows - j < window) | (j < sinks))
        clean, _, t = attended(q, k, v, d ** -0.5, window, sinks)
        first = slice(0, heads // kv)  # the heads of key head 0
        hidden = torch.ones(n, heads, dtype=torch.bool)
        hidden[see, first] = False
        got = out.cpu().double()
        assert bool(torch.isfinite(got[hidden]).all())
        assert bool(((got - clean).abs() <= t)[hidden].all())
        if x is v:
            col = got[see][:, first, d // 2]
            assert not bool(torch.isfinite(col).any())
            rest = torch.ones(d, dtype=torch.bool)
            rest[d // 2] = False
            assert bool(torch.isfinite(got[see][:, first][..., rest]).all())
        elif math.isnan(bad):
            assert bool(torch.isnan(got[see][:, first]).all())


def test_large_scores(ctx):
    """Scores far apart: the running maximum carries the sums."""
    cache, seqs = filled(ctx, [500], 16, 1, 64, F32, seed=4)
    cache.k.mul_(30.0)
    kk = seqs[0][0] * 30.0
    q = normal(gen(10), 1, 2, 64) * 30.0
    out = cache.attend(q)
    o, _, t = attended(q, kk[0], seqs[0][1][0], 0.125, None, 0)
    check(out, o, t)


@pytest.mark.parametrize("dtype,d,r,layout", [(BF, 128, 128, "half"), (F16, 96, 48, "interleaved"),
                                              (F32, 37, 10, "half")])
@pytest.mark.parametrize("order", ["nhd", "hnd"])
def test_append(ctx, dtype, d, r, layout, order):
    """The new tokens' rows land in their places, turned; no other row of the
    pool changes."""
    from vectorstorekit_amd import RotaryEmbedding

    lengths, news, page, kv, heads = [40, 7, 16, 100], [40, 1, 0, 33], 16, 2, 6
    cache, _ = filled(ctx, lengths, page, kv, d, dtype, layers=2, order=order, seed=d,
                      poison=False)
    rope = RotaryEmbedding(ctx, d, rotary_dim=r, layout=layout)
    starts = [0] + list(np.cumsum(news))
    g = gen(11)
    q, k, v = (normal(g, starts[-1], h, d, dtype=dtype) for h in (heads, kv, kv))
    want_k, want_v = cache.k.cpu().clone(), cache.v.cpu().clone()
    table = cache.table.cpu()
    pos = torch.cat([torch.arange(L - n, L) for L, n in zip(lengths, news)]).to(torch.int32).to(DEV)
    turned_q, turned_k = rope.apply(q, k, positions=pos)
    out = cache.append(k, v, starts=starts, max_new=40, layer=1, rotary=rope, q=q)
    assert torch.equal(out, turned_q)
    t = 0
    for s, (length, n) in enumerate(zip(lengths, news)):
        for p in range(length - n, length):
            want_k[1, table[s, p // page], p % page] = turned_k[t].cpu()
            want_v[1, table[s, p // page], p % page] = v[t].cpu()
            t += 1
    assert torch.equal(cache.k.cpu(), want_k) and torch.equal(cache.v.cpu(), want_v)
    # one token each, slots out of order, as it is
    k1, v1 = normal(g, 2, kv, d, dtype=dtype), normal(g, 2, kv, d, dtype=dtype)
    assert cache.append(k1, v1, seqs=[3, 0]) is None
    for i, s in enumerate((3, 0)):
        p = lengths[s] - 1
        want_k[0, table[s, p // page], p % page] = k1[i].cpu()
        want_v[0, table[s, p // page], p % page] = v1[i].cpu()
    assert torch.equal(cache.k.cpu(), want_k) and torch.equal(cache.v.cpu(), want_v)


# ---------------------------------------------------------------------- the pages

class Model:
    """The page keeping on the host: lists and a loop."""

    def __init__(self, cache):
        self.page, self.width = cache.page_size, cache.width
        self.k, self.v = cache.k.cpu().clone(), cache.v.cpu().clone()
        self.table = cache.table.cpu().tolist()
        self.lengths, self.refs = cache.lengths.cpu().tolist(), cache.refs.cpu().tolist()

    def take(self, left):
        return next((i for i, r in enumerate(self.refs) if r == 0), None) if left else None

    def free(self, seqs):
        for s in seqs:
            for i, p in enumerate(self.table[s]):
                if p >= 0:
                    self.refs[p] -= 1
                self.table[s][i] = -1
            self.lengths[s] = 0

    def reserve(self, seqs, counts):
        missing = 0
        for s, n in zip(seqs, counts):
            old, to = self.lengths[s], self.lengths[s] + n
            for i in range(-(-old // self.page), -(-to // self.page)):
                p = self.take(i < self.width)
                if p is None:
                    missing += 1
                    to = min(to, i * self.page)
                else:
                    self.table[s][i], self.refs[p] = p, 1
            self.lengths[s] = to
        return missing

    def fork(self, parents, children):
        missing = 0
        self.free(children)
        for f, c in zip(parents, children):
            for i in range(self.lengths[f] // self.page):
                self.table[c][i] = self.table[f][i]
                self.refs[self.table[f][i]] += 1
        for f, c in zip(parents, children):
            full, fill = divmod(self.lengths[f], self.page)
            self.lengths[c] = full * self.page
            if fill:
                p = self.take(True)
                if p is None:
                    missing += 1
                    continue
                self.table[c][full], self.refs[p] = p, 1
                for x in (self.k, self.v):
                    x[:, p, :fill] = x[:, self.table[f][full], :fill]
                self.lengths[c] += fill
        return missing

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [i for i in range(live) if self.refs[i] == 0]
        movers = [i for i in range(live, len(self.refs)) if self.refs[i] > 0]
        for to, at in zip(holes, movers):
            for x in (self.k, self.v):
                x[:, to] = x[:, at]
            self.refs[to], self.refs[at] = self.refs[at], 0
        new = dict(zip(movers, holes))
        self.table = [[new.get(p, p) for p in row] for row in self.table]
        return live

    def same(self, cache):
        assert cache.table.cpu().tolist() == self.table
        assert cache.lengths.cpu().tolist() == self.lengths
        assert cache.refs.cpu().tolist() == self.refs
        assert torch.equal(cache.k.cpu(), self.k) and torch.equal(cache.v.cpu(), self.v)


@pytest.mark.parametrize("dtype,kv,d,order", [(BF, 2, 64, "nhd"), (F16, 3, 5, "nhd"),
                                              (F32, 2, 32, "hnd"), (F16, 2, 3, "hnd")])
@pytest.mark.parametrize("pages", [40, 5000])
def test_pages(ctx, dtype, kv, d, order, pages):
    """A program's life: sequences grow, branch, end and the pool is packed,
    step by step as on the host; with 40 pages it runs out of them."""
    from vectorstorekit_amd import PagedKVCache

    page, slots, width, layers = 16, 8, 9, 2
    g = gen(pages + d)
    shape = (layers, pages, page, kv, d)
    k, v = (torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(2))
    if order == "hnd":
        k, v = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in (k, v))
    refs = torch.zeros(pages, dtype=torch.int32)
    if pages > 100:  # most of a large pool is held by others
        refs[torch.randperm(pages, generator=g)[: pages - 60]] = 1
    cache = PagedKVCache.over(ctx, k, v, torch.full((slots, width), -1, dtype=torch.int32,
                                                    device=DEV),
                              torch.zeros(slots, dtype=torch.int32, device=DEV), refs.to(DEV))
    m = Model(cache)
    rng = np.random.default_rng(pages)
    short = 0
    for step in range(40):
        what = rng.integers(0, 5)
        if what <= 1:
            seqs = rng.permutation(slots)[: rng.integers(1, slots + 1)].tolist()
            counts = rng.integers(0, 50, len(seqs)).tolist()
            missing = m.reserve(seqs, counts)
            cache.reserve(seqs, counts)
            assert cache.missing() == missing
            short += missing
        elif what == 2:
            order_ = rng.permutation(slots).tolist()
            n = int(rng.integers(1, slots // 2 + 1))
            children = order_[:n]
            parents = [order_[n + int(rng.integers(0, slots - n))] for _ in range(n)]
            missing = m.fork(parents, children)
            cache.fork(parents, children)
            assert cache.missing() == missing
            short += missing
        elif what == 3:
            seqs = rng.permutation(slots)[: rng.integers(0, 3)].tolist()
            m.free(seqs)
            cache.free(seqs)
        else:
            assert int(cache.compact()) == m.compact()
        m.same(cache)
    assert short > 0 or pages > 100


@pytest.mark.parametrize("slots,width", [(32, 4), (33, 1 << 26)])
def test_reserve_more_than_32_bits_of_pages(ctx, slots, width):
    """Pages wanted in all pass 2^31: they are counted as far as that, and the
    first sequences get what there is."""
    from vectorstorekit_amd import PagedKVCache

    cache = PagedKVCache(ctx, pages=40, page_size=16, kv_heads=1, head_dim=8, slots=slots,
                         width=width, dtype=F16)
    cache.reserve(list(range(slots)), [2 ** 31 - 1] * slots)
    assert cache.missing() == 2 ** 31 - 1
    each = min(width, 40)
    want = [16 * max(0, min(each, 40 - i * each)) for i in range(slots)]
    assert cache.lengths.tolist() == want
    assert cache.refs.tolist() == [1] * 40
    for i, n in enumerate(want):
        assert cache.table[i, :n // 16].tolist() == list(range(i * each, i * each + n // 16))
        assert bool((cache.table[i, n // 16:] == -1).all())


@pytest.mark.parametrize("pages", [3500, 33000])
def test_fork_many(ctx, pages):
    """More branches than a workgroup has threads, twice: the second drops the
    first's; with 3,500 pages some find no last page."""
    from vectorstorekit_amd import PagedKVCache

    page, slots, width, roots = 16, 1700, 3, 200
    g = gen(pages)
    k, v = (torch.randn((1, pages, page, 1, 4), generator=g).to(F16).to(DEV) for _ in range(2))
    refs = (torch.rand(pages, generator=g) < 0.55).int()  # held by others
    cache = PagedKVCache.over(ctx, k, v, torch.full((slots, width), -1, dtype=torch.int32,
                                                    device=DEV), ints([0] * slots), refs.to(DEV))
    m = Model(cache)
    rng = np.random.default_rng(pages)
    counts = rng.integers(0, page * width + 1, roots).tolist()
    assert m.reserve(range(roots), counts) == 0
    cache.reserve(list(range(roots)), counts)
    for _ in range(2):
        children = (roots + rng.permutation(slots - roots)).tolist()
        parents = rng.integers(0, roots, len(children)).tolist()
        missing = m.fork(parents, children)
        cache.fork(parents, children)
        assert cache.missing() == missing
        assert (missing > 0) == (pages < 10000)
        m.same(cache)


def test_copy_pages(ctx):
    cache, _ = filled(ctx, [100], 32, 2, 40, F16, layers=3, seed=1, poison=False)
    k, v = cache.k.cpu().clone(), cache.v.cpu().clone()
    cache.copy_pages([0, 2], [5, 4])
    for x in (k, v):
        x[:, [5, 4]] = x[:, [0, 2]]
    assert torch.equal(cache.k.cpu(), k) and torch.equal(cache.v.cpu(), v)


# ------------------------------------------------------------- streams and graphs

def test_other_stream_and_graph(ctx):
    """A decoding step on a stream of its own, captured and replayed with new
    inputs: each replay equals the eager calls."""
    from vectorstorekit_amd import RotaryEmbedding

    cache, _ = filled(ctx, [700, 33], 32, 2, 64, BF, seed=12, poison=False)
    rope = RotaryEmbedding(ctx, 64)
    q, k, v = (torch.zeros(2, h, 64, dtype=BF, device=DEV) for h in (4, 2, 2))

    def step():
        turned = cache.append(k, v, rotary=rope, q=q)
        return cache.attend(turned, window=300, sinks=4)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        g = gen(20 + i)
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g).to(BF))
        graph.replay()
        got = held.clone()
        eager = step()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


# ------------------------------------------------------------------------ refusals

# -------------------------------------------- many rows: tiles of 128 query rows

def attended_at_once(q, k, v, scale, window, sinks):
    """``attended``, all heads and tokens in one product."""
    t, heads, d = q.shape
    u = U[q.dtype]
    q, k, v = (x.detach().cpu().double().transpose(0, 1) for x in (q, k, v))
    length, group = k.shape[1], heads // k.shape[0]
    if t == 0 or length == 0:
        zero = torch.zeros(t, heads, d, dtype=torch.float64)
        return zero, torch.full((t, heads), -math.inf, dtype=torch.float64), zero
    k, v = (x.repeat_interleave(group, 0) for x in (k, v))
    j, pos = torch.arange(length)[None], torch.arange(length - t, length)[:, None]
    see = j <= pos
    if window:
        see = see & ((pos - j < window) | (j < sinks))
    some = see.any(1)[None, :, None]
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, 2)
    w = torch.exp(s - lse[..., None].masked_fill(~some, 0.0)).masked_fill(~see, 0.0)
    out = w @ v
    products = (q.abs() @ k.abs().transpose(1, 2)).masked_fill(~see, 0.0)
    e = 2.0 ** -24 * (d + 8) * scale * products.amax(2, keepdim=True)
    peak = torch.where(see[None], v.abs().amax(2)[:, None], 0.0).amax(2, keepdim=True)
    tol = u * out.abs() + peak * (2 * (e + 2.0 ** -21 + 2.0 ** -24 * (length + 16)) + u)
    return out.transpose(0, 1), lse.transpose(0, 1), tol.transpose(0, 1)


def kernels_of(ctx, f):
    ctx.profile_reset()
    ctx.profile(True)
    try:
        out = f()
        return out, set(ctx.profile_stats())
    finally:
        ctx.profile(False)
        ctx.profile_reset()


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("order", ["nhd", "hnd"])
@pytest.mark.parametrize("news,lengths,page,heads,kv,d,window,sinks", [
    ([70, 130], [200, 130], 32, 64, 8, 128, 33, 4),
    ([65, 64, 63], [65, 100, 63], 16, 96, 96, 64, 16, 16),
    ([300], [300], 64, 32, 4, 96, 64, 0),
    ([40, 9, 0], [64, 20, 5], 16, 80, 10, 256, None, 0),
    ([260], [900], 64, 36, 9, 80, 200, 70),    # the sinks' last tile holds window too
    ([129], [1500], 16, 64, 8, 128, 300, 17),
    ([1, 512], [1, 512], 16, 16, 2, 40, 100, 1),
    ([150], [1000], 128, 60, 20, 256, 333, 40),
    ([64], [20000], 64, 8, 1, 128, None, 0),   # few rows, many keys: in parts
    ([64], [9000], 32, 16, 2, 256, None, 0),
    ([64], [9000], 32, 16, 16, 64, 8500, 3),
])
def test_prompt_attention_of_many_rows(ctx, dtype, order, news, lengths, page, heads, kv, d,
                                       window, sinks):
    cache, seqs = filled(ctx, lengths, page, kv, d, dtype, order=order, seed=d + 2)
    starts = [0] + list(np.cumsum(news))
    q = normal(gen(11), starts[-1], heads, d, dtype=dtype)
    (out, lse), used = kernels_of(ctx, lambda: cache.attend(
        q, starts=starts, max_new=max(news), window=window, sinks=sinks, return_lse=True))
    assert "attn_tile" in used
    for i, (kk, vv) in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        o, l, t = attended_at_once(q[a:b], kk[0], vv[0], d ** -0.5, window, sinks)
        check(out[a:b], o, t)
        check_norm(out[a:b], o, dtype)
        check(lse[a:b], l, 2.0 ** -16 * (1 + l.abs()))


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("lengths,heads,kv,d,window,sinks", [
    ([520, 31], 8, 2, 128, 100, 130),
    ([333, 0, 1], 24, 24, 64, 90, 5),
    ([130], 64, 64, 128, None, 0),
    ([190, 75], 32, 4, 256, 32, 0),
    ([1030], 8, 8, 96, 64, 4),
    ([500], 33, 11, 72, 1, 1),
])
def test_window_attention_of_many_rows(ctx, dtype, lengths, heads, kv, d, window, sinks):
    from vectorstorekit_amd import window_attention

    starts = [0] + list(np.cumsum(lengths))
    packed = normal(gen(d + 3), starts[-1], heads + 2 * kv, d, dtype=dtype)
    q, k, v = packed[:, :heads], packed[:, heads:heads + kv], packed[:, heads + kv:]
    (out, lse), used = kernels_of(ctx, lambda: window_attention(
        ctx, q, k, v, starts=starts, max_length=max(lengths), window=window, sinks=sinks,
        return_lse=True))
    assert "attn_tile" in used
    for i in range(len(lengths)):
        a, b = starts[i], starts[i + 1]
        o, l, t = attended_at_once(q[a:b], k[a:b], v[a:b], d ** -0.5, window, sinks)
        check(out[a:b], o, t)
        check_norm(out[a:b], o, dtype)
        check(lse[a:b], l, 2.0 ** -16 * (1 + l.abs()))


def test_many_queries_before_the_keys(ctx):
    from vectorstorekit_amd import window_attention

    q, k, v = (normal(gen(12), n, 32, 64, dtype=BF) for n in (300, 250, 250))
    out, lse = window_attention(ctx, q, k, v, starts=[0, 290, 300], k_starts=[0, 250, 250],
                                return_lse=True)
    assert not out[:40].any() and not out[290:].any()
    assert bool(torch.isneginf(lse[:40]).all()) and bool(torch.isneginf(lse[290:]).all())
    o, _, t = attended_at_once(q[40:290], k, v, 64 ** -0.5, None, 0)
    check(out[40:290], o, t)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,kv,d,n", [(64, 32, 128, 150), (48, 48, 64, 400),
                                          (128, 16, 256, 70)])
def test_masked_places_of_many_rows(ctx, dtype, bad, heads, kv, d, n):
    """As above, and a hidden key between the sinks and the window."""
    from vectorstorekit_amd import window_attention

    g = gen(13)
    q, k, v = (normal(g, n, h, d, dtype=dtype) for h in (heads, kv, kv))
    window, sinks = 20, 3
    clean, _, t = attended_at_once(q, k, v, d ** -0.5, window, sinks)
    for x, j in ((k, n - 45), (v, n - 45), (v, 1), (v, 7), (k, 7)):
        y = [z.clone() for z in (k, v)]
        (y[0] if x is k else y[1])[j, 0, d // 2] = bad
        out = window_attention(ctx, q, *y, starts=[0, n], window=window, sinks=sinks)
        rows = torch.arange(n)
        see = (rows >= j) & ((rows - j < window) | (j < sinks))
        first = slice(0, heads // kv)
        hidden = torch.ones(n, heads, dtype=torch.bool)
        hidden[see, first] = False
        got = out.cpu().double()
        assert bool(((got - clean).abs() <= t)[hidden].all())
        if x is v:
            assert not bool(torch.isfinite(got[see][:, first, d // 2]).any())
            rest = torch.ones(d, dtype=torch.bool)
            rest[d // 2] = False
            assert bool(((got - clean).abs() <= t)[see][:, first][..., rest].all())
        elif math.isnan(bad):
            assert bool(torch.isnan(got[see][:, first]).all())


def test_example(capsys):
    """The example's decoder over the cache against itself without one.  Both
    round activations to bf16 at the same places, in another order of sums:
    eight roundings a layer of 2^-8 of a value, four layers, added as
    independent errors, are 2^-8 sqrt(32) = 0.022 of a logit's size, twice
    that for the largest of them."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "answer_over_retrieved.py")
    spec = importlib.util.spec_from_file_location("answer_over_retrieved", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(branches=3, steps=6) <= 0.044
    assert "documents [123" in capsys.readouterr().out


def test_offsets_out_of_order(ctx):
    """Offsets that fall, as far apart as 32 bits allow: no token is treated."""
    for starts in ([2 ** 31 - 1, -2 ** 31], [5, 2], [9, 9]):
        cache, _ = filled(ctx, [40], 16, 2, 64, BF, poison=False)
        k, v = cache.k.clone(), cache.v.clone()
        x = normal(gen(3), 8, 2, 64, dtype=BF)
        cache.append(x, x, starts=ints(starts), seqs=ints([0]))
        cache.attend(x, starts=ints(starts), seqs=ints([0]))
        torch.cuda.synchronize()
        assert torch.equal(cache.k, k) and torch.equal(cache.v, v)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new,lengths", [(1, [900] * 12), (3, [7000, 20, 0, 300]), (80, [2000, 90])])
def test_bound_of_dense_keys(ctx, dtype, new, lengths):
    """It only divides the work, wrong ones included."""
    from vectorstorekit_amd import window_attention

    g, n = gen(new), len(lengths)
    ks, starts = [0] + list(np.cumsum(lengths)), list(range(0, n * new + 1, new))
    q, k, v = (normal(g, m, h, 64, dtype=dtype) for m, h in ((n * new, 8), (ks[-1], 2), (ks[-1], 2)))
    for bound in (None, max(lengths), 1, 10 ** 6):
        out = window_attention(ctx, q, k, v, starts=ints(starts), k_starts=ints(ks), max_length=new,
                               max_keys=bound)
        for i in range(n):
            a, b = starts[i], starts[i + 1]
            o, _, t = attended_at_once(q[a:b], k[ks[i]:ks[i + 1]], v[ks[i]:ks[i + 1]], 0.125, None, 0)
            check(out[a:b], o, t)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv,d,news,most", [(4, 2, 64, [9, 3, 1], 4), (32, 8, 128, [200, 70], 96),
                                                  (6, 6, 100, [40, 2], 1)])
def test_bound_under_the_new_tokens(ctx, dtype, heads, kv, d, news, most):
    """A sequence's first max_new rows are treated, each at its own place."""
    lengths = [x + 50 for x in news]
    cache, seqs = filled(ctx, lengths, 16, kv, d, dtype, seed=d)
    starts = [0] + list(np.cumsum(news))
    q = normal(gen(3), starts[-1], heads, d, dtype=dtype)
    out, lse = cache.attend(q, starts=starts, max_new=most, window=60, sinks=2, return_lse=True)
    k = cache.k.clone()
    x = normal(gen(4), starts[-1], kv, d, dtype=dtype)
    cache.append(x, x, starts=starts, max_new=most)
    for i, (kk, vv) in enumerate(seqs):
        a, n = starts[i], min(news[i], most)
        o, l, t = attended_at_once(q[a:starts[i + 1]], kk[0], vv[0], d ** -0.5, 60, 2)
        check(out[a:a + n], o[:n], t[:n])
        check(lse[a:a + n], l[:n], 2.0 ** -16 * (1 + l[:n].abs()))
        for p in range(lengths[i]):
            page, row = int(cache.table[i, p // 16]), p % 16
            new = p - 50
            want = x[a + new] if 0 <= new < n else k[0, page, row]
            assert torch.equal(cache.k[0, page, row], want)


@pytest.mark.parametrize("d,lengths", [(64, [20]), (128, [9000]), (256, [70, 30])])
def test_no_rows_to_treat(ctx, d, lengths):
    """Bounds of no new token at all: nothing is done, however long the keys."""
    from vectorstorekit_amd import window_attention

    cache, seqs = filled(ctx, lengths, 16, 2, d, BF, width=600, seed=d)
    starts = [0] + list(range(1, len(lengths) + 1))
    q = normal(gen(d), len(lengths), 4, d, dtype=BF)
    out, lse = cache.attend(q, starts=starts, max_new=0, return_lse=True)
    assert out.shape == q.shape and lse.shape == q.shape[:2]
    k = cache.k.clone()
    cache.append(q[:, :2], q[:, 2:], starts=starts, max_new=0)
    assert torch.equal(cache.k.view(torch.int16), k.view(torch.int16))
    x = normal(gen(1), 5000, 2, d, dtype=BF)
    assert window_attention(ctx, x, x, x, starts=[0, 5000], max_length=0).shape == x.shape
    assert cache.attend(q[:0], starts=[0], max_new=0).shape == (0, 4, d)
    # and the calls after them are as ever
    out = cache.attend(q, starts=starts, max_new=1)
    for i, (kk, vv) in enumerate(seqs):
        o, _, t = attended(q[i:i + 1], kk[0], vv[0], d ** -0.5, None, 0)
        check(out[i:i + 1], o, t)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("new,n", [(1, 100003), (1, 900), (2, 6000), (70, 20000)])
def test_small_weights_of_many_keys(ctx, dtype, new, n):
    """One first key of value 0 takes nearly all of a row's weight; the others,
    2^-27 each, are the whole output: w (n - 1) / (1 + w (n - 1)) of them.
    Scores are sums of products of powers of two, so they are exact: the weight
    is off by 2^-21, the sum of n by 2^-24 (n + 16) at the most, an f16 or bf16
    weight and output by u each (an f16 output under 2^-14 by 2^-25)."""
    from vectorstorekit_amd import window_attention

    heads, d = 32, 64
    k = torch.zeros(n, heads, d, dtype=dtype, device=DEV)
    v = torch.ones(n, heads, d, dtype=dtype, device=DEV)
    k[0, :, 0], v[0] = 32.0, 0.0
    q = torch.zeros(new, heads, d, dtype=dtype, device=DEV)
    q[:, :, 0] = 32.0
    scale = 27 * math.log(2) / 1024
    out, lse = window_attention(ctx, q, k, v, starts=[0, new], k_starts=[0, n], scale=scale,
                                return_lse=True)
    # (the scale as the call takes it, in fp32)
    w = math.exp(-1024 * float(np.float32(scale)))
    others = w * torch.arange(n - new, n, dtype=torch.float64)[:, None, None]
    want = (others / (1 + others)).expand(new, heads, d)
    u = U[dtype] if dtype != F32 else 0.0
    # (the first score, 27 in log2, is rounded twice to 2^-20 of it: 2^-19 of w)
    tol = want * (2 * U[dtype] + u + 2 * 2.0 ** -19 + 2.0 ** -24 * (n + 16)) + 2.0 ** -25
    check(out, want, tol if dtype == F16 else tol - 2.0 ** -25)
    top = 1024 * float(np.float32(scale))
    check(lse, (top + torch.log1p(others))[..., 0].expand(new, heads),
          torch.full((new, heads), 2.0 ** -16 * 28, dtype=torch.float64))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("new,n", [(1, 60), (1, 40003), (3, 500), (70, 300), (70, 20000), (600, 700)])
@pytest.mark.parametrize("scale", [0.2, 0.9, 3.7, 1e3, 1e6])
def test_scores_that_differ_by_one_rounding(ctx, dtype, new, n, scale):
    """Scores of +-2^24 and more times ``scale``: in 32 bits a softmax of such
    scores is the mean over the largest, which many keys share here.  Scores
    are one product of two values, exact in fp32, so the weights are 1 (off by
    2^-21 at the most) and 0; the sum, weight and output are as above."""
    from vectorstorekit_amd import window_attention

    heads, d = 32, 64
    g = gen(n + new)
    k = torch.zeros(n, heads, d)
    # large negative ones first, then, for some of the heads, larger ones, and
    # zeros for the last: the running maximum climbs as far as it can
    k[:, :, 0] = torch.where(torch.rand(n, heads, generator=g) < 0.3, -1168.0, -1200.0)
    later = torch.arange(n)[:, None] >= n // 2
    some = torch.rand(n, heads, generator=g) < 0.4
    k[:, 8:16, 0] = torch.where(later & some, 1168.0, k[:, :, 0])[:, 8:16]
    k[:, 16:24, 0] = torch.where(later & some, 1e-3, k[:, :, 0])[:, 16:24]
    k[:, 24:, 0] = k[:, 24:, 0].neg()
    k, v = k.to(dtype).to(DEV), normal(g, n, heads, d, dtype=dtype)
    q = torch.zeros(new, heads, d, dtype=dtype, device=DEV)
    q[:, :, 0] = 14592.0  # 57 * 2^8
    out, lse = window_attention(ctx, q, k, v, starts=[0, new], k_starts=[0, n], scale=scale,
                                return_lse=True)
    u = U[dtype]
    rows = [0, 1, new // 2, new - 1]
    for i in sorted(set(r for r in rows if r < new)):
        m = n - new + i + 1
        s = q[i, :, :1].cpu().double() * k[:m, :, 0].cpu().double().T  # heads x keys
        s *= float(np.float32(scale))
        w = torch.softmax(s, 1)
        vv = v[:m].cpu().double()
        want = torch.einsum("hm,mhd->hd", w, vv)
        tol = u * want.abs() + float(vv.abs().max()) * (
            2 * (2.0 ** -21 + 2.0 ** -24 * (n + 16)) + (u if dtype != F32 else 0))
        check(out[i], want, tol)
        le = torch.logsumexp(s, 1)
        check(lse[i], le, 2.0 ** -16 + 2.0 ** -21 * s.abs().amax(1))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("heads,kv,d,new,n", [(8, 2, 128, 1, 700), (8, 8, 64, 1, 90),
                                              (4, 1, 256, 1, 9000), (6, 3, 100, 1, 300),
                                              (4, 2, 128, 40, 300), (5, 5, 33, 20, 130),
                                              (64, 32, 128, 130, 300), (48, 48, 64, 400, 400),
                                              (128, 16, 256, 70, 200)])
def test_infinite_values(ctx, dtype, heads, kv, d, new, n):
    """A visible infinity is the sum of its column, with its sign; two of
    different signs are NaN; a row that does not see it is as without it.  The
    weight is an ordinary one, and one of 2^-40 of the largest."""
    from vectorstorekit_amd import window_attention

    g = gen(d + new)
    q, k, v = (normal(g, m, h, d, dtype=dtype) for m, h in ((new, heads), (n, kv), (n, kv)))
    window, sinks = n - new // 2, 3
    # key 5 of key head 1 has a score 40 in log2 below every other's largest
    low = 1 if kv > 1 else 0
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[5, low] = 0.0
    k[5, low, 0] = -64.0
    scale = 40 * math.log(2) / 512
    clean, _, t = attended_at_once(q, k, v, scale, window, sinks)
    for where in ([(n - new, 1.0)], [(2, -1.0)], [(5, 1.0)], [(n - new, 1.0), (n // 2, -1.0)]):
        bad, want = v.clone(), clean.clone()
        for j, sign in where:
            bad[j, low, d // 2] = sign * math.inf
        for i in range(new):
            pos = n - new + i
            signs = {sign for j, sign in where if j <= pos and (pos - j < window or j < sinks)}
            if signs:
                one = slice(low * (heads // kv), (low + 1) * (heads // kv))
                want[i, one, d // 2] = math.nan if len(signs) > 1 else signs.pop() * math.inf
        out = window_attention(ctx, q, k, bad, starts=[0, new], k_starts=[0, n], scale=scale,
                               window=window, sinks=sinks).cpu().double()
        odd = ~torch.isfinite(want)
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        assert torch.equal(out[torch.isinf(want)], want[torch.isinf(want)])
        check(out.masked_fill(odd, 0.0), want.masked_fill(odd, 0.0), t.masked_fill(odd, 0.0))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("heads,kv,d,news,lengths", [
    (8, 2, 128, [1, 1], [300, 41]), (8, 8, 64, [1], [20000]), (6, 3, 100, [1, 1], [90, 500]),
    (4, 2, 64, [20, 3], [130, 33]), (64, 16, 128, [140, 70], [300, 80]),
    (32, 8, 256, [90], [200]), (8, 8, 64, [64], [20000]),
])
def test_key_by_key_over_pages(ctx, dtype, heads, kv, d, news, lengths):
    """Scores that differ by one rounding and infinite values in a paged cache
    whose other places hold NaN: as over dense keys."""
    from vectorstorekit_amd import window_attention

    cache, seqs = filled(ctx, lengths, 32, kv, d, dtype, seed=heads + d)
    g = gen(d)
    starts = [0] + list(np.cumsum(news))
    kstarts = [0] + list(np.cumsum(lengths))
    k, v = (torch.cat([x[i][0] for x in seqs]) for i in (0, 1))
    # a few of each sequence's keys have the largest score, and one value is
    # infinite
    k[:], best = 0.0, torch.rand(k.shape[:2], generator=g) < 0.2
    k[..., 0] = torch.where(best, -1168.0, -1200.0).to(dtype)
    for a in kstarts[:-1]:
        k[a, :, 0] = -1168.0
    odd = [a + 7 for a in kstarts[:-1]]
    k[odd, :, 0] = -1168.0
    peak = float(v.abs().max())
    v[odd, 0, d // 2] = math.inf
    q = torch.zeros(starts[-1], heads, d, dtype=dtype, device=DEV)
    q[:, :, 0] = 14592.0
    table = cache.table.cpu()
    for i, n in enumerate(lengths):
        for p in range(0, n, 32):
            page, m, at = int(table[i, p // 32]), min(32, n - p), kstarts[i] + p
            cache.k[0, page, :m], cache.v[0, page, :m] = k[at:at + m].to(DEV), v[at:at + m].to(DEV)
    for scale in (3.7, 1e6):
        given = {"scale": scale, "window": 10 ** 6, "sinks": 0, "return_lse": True}
        out, lse = cache.attend(q, starts=starts, max_new=max(news), **given)
        same, also = window_attention(ctx, q, k.to(DEV), v.to(DEV), starts=starts, k_starts=kstarts,
                                      **given)
        for i, n in enumerate(lengths):
            for t in {0, news[i] // 2, news[i] - 1}:
                r, m = starts[i] + t, n - news[i] + t + 1
                s = q[r, :, :1].cpu().double() * k[kstarts[i]:kstarts[i] + m].repeat_interleave(
                    heads // kv, 1)[..., 0].double().T * float(np.float32(scale))
                w = torch.softmax(s, 1)
                vv = v[kstarts[i]:kstarts[i] + m].double().repeat_interleave(heads // kv, 1)
                want = torch.where(w.T[..., None] > 0, w.T[..., None] * vv, 0.0).sum(0)
                u = U[dtype]
                tol = u * want.abs() + peak * (2 * (2.0 ** -21 + 2.0 ** -24 * (n + 16))
                                               + (u if dtype != F32 else 0))
                inf = torch.isinf(want)
                for x, y in ((out[r], lse[r]), (same[r], also[r])):
                    x = x.cpu().double()
                    assert torch.equal(x[inf], want[inf])
                    check(x.masked_fill(inf, 0.0), want.masked_fill(inf, 0.0),
                          tol.masked_fill(inf, 0.0))
                    check(y, torch.logsumexp(s, 1), 2.0 ** -16 + 2.0 ** -21 * s.abs().amax(1))


def test_refusals_of_lost_meaning(ctx):
    """What would otherwise pass and mean something else."""
    from vectorstorekit_amd import RotaryEmbedding, VSKError, window_attention

    def refused(kind, f, *a, **k):
        with pytest.raises(VSKError) as e:
            f(*a, **k)
        assert e.value.kind == kind, e.value

    cache, _ = filled(ctx, [20, 4], 16, 2, 64, F32, poison=False)
    x, pos = torch.ones(2, 2, 64, device=DEV), ints([0, 1])
    rope = RotaryEmbedding(ctx, 64)
    rope.free()  # (not "no rotation")
    refused("invalidArgument", cache.append, x, x, rotary=rope)
    refused("invalidArgument", rope.apply, x, positions=pos)
    for far in (1 << 32, -(1 << 32), 1 << 31):  # (not slot 0)
        refused("invalidArgument", cache.free, [far])
        refused("invalidArgument", cache.reserve, [0], [far])
    assert cache.lengths.tolist() == [20, 4]
    rope, y = RotaryEmbedding(ctx, 64), x.clone().requires_grad_()
    refused("unsupportedOperation", rope.apply, y, positions=pos)
    refused("unsupportedOperation", cache.attend, y)
    refused("unsupportedOperation", cache.append, x, y)
    refused("unsupportedOperation", window_attention, ctx, x, y, x, starts=[0, 2])
    with torch.no_grad():
        assert torch.equal(rope.apply(y, positions=pos), rope.apply(x, positions=pos))
        assert torch.equal(cache.attend(y), cache.attend(x))


def test_tangents_are_refused(ctx):
    """Forward-mode and functional gradients are not dropped silently."""
    from torch.autograd import forward_ad

    from vectorstorekit_amd import RotaryEmbedding, VSKError, window_attention

    cache, _ = filled(ctx, [20, 4], 16, 2, 64, F32, poison=False)
    x, pos, rope = torch.ones(2, 2, 64, device=DEV), ints([0, 1]), RotaryEmbedding(ctx, 64)
    calls = (lambda y: rope.apply(y, positions=pos), cache.attend,
             lambda y: cache.append(x, y), lambda y: cache.append(x, x, q=y),
             lambda y: window_attention(ctx, x, y, x, starts=[0, 2]))
    for grads in (True, False):
        with forward_ad.dual_level(), torch.set_grad_enabled(grads):
            for f in calls:
                with pytest.raises(VSKError) as e:
                    f(forward_ad.make_dual(x, x))
                assert e.value.kind == "unsupportedOperation"
            rope.apply(x, positions=pos)  # one without a tangent is as ever
    for f in calls:
        with pytest.raises((VSKError, RuntimeError)):
            torch.func.jvp(f, (x,), (x,))
        with pytest.raises((VSKError, RuntimeError)):
            torch.func.vjp(f, x)


def test_expanded_tensors_are_not_turned_in_place(ctx):
    """Tokens (or heads) at one place would be turned once each, one after
    another, or not; out of place they are read only."""
    from vectorstorekit_amd import RotaryEmbedding, VSKError

    rope, pos = RotaryEmbedding(ctx, 64), ints(range(1, 8))
    one, head = normal(gen(1), 1, 2, 64), normal(gen(2), 7, 1, 64)
    x = normal(gen(3), 7, 2, 64)
    for y in (one.expand(7, 2, 64), head.expand(7, 2, 64)):
        before = y.clone()
        for q, k in ((y, None), (y, x.clone()), (x.clone(), y)):
            with pytest.raises(VSKError) as e:
                rope.apply(q, k, positions=pos, inplace=True)
            assert e.value.kind == "invalidArgument"
        assert torch.equal(y, before)
        assert torch.equal(rope.apply(y, positions=pos), rope.apply(before, positions=pos))
    z = one.clone().expand(1, 2, 64)
    assert torch.equal(rope.apply(z, positions=pos[:1], inplace=True),
                       rope.apply(one, positions=pos[:1]))


def off_by_one(x):
    """x's values one element past an aligned place."""
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
    y = flat[1:].view(x.shape)
    return y.copy_(x)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d,shift", [(68, 0), (100, 0), (101, 0), (77, 0), (128, 1), (64, 1),
                                     (256, 1), (250, 0)])
@pytest.mark.parametrize("news,lengths,heads,kv,window,sinks", [
    ([1, 1, 1], [700, 1, 0], 8, 2, None, 0),
    ([1], [5000], 5, 5, 900, 3),
    ([1] * 40, [60 + i for i in range(40)], 6, 1, 33, 1),
    ([40, 3, 0, 90], [300, 3, 9, 90], 6, 3, 50, 2),
    ([200, 150], [200, 150], 4, 4, None, 0),
    ([100] * 6, [100] * 6, 32, 8, 70, 5),  # a wave a row tile
])
def test_operands_without_wide_loads(ctx, dtype, d, shift, news, lengths, heads, kv, window, sinks):
    """Heads that are not whole 16-byte pieces, and bases off by an element:
    tokens, prompts and dense keys."""
    from vectorstorekit_amd import PagedKVCache, window_attention

    cache, seqs = filled(ctx, lengths, 16, kv, d, dtype, seed=d + shift)
    if shift:
        cache = PagedKVCache.over(ctx, off_by_one(cache.k), off_by_one(cache.v), cache.table,
                                  cache.lengths)
    starts = [0] + list(np.cumsum(news))
    q = normal(gen(d), starts[-1], heads, d, dtype=dtype)
    given = {"window": window, "sinks": sinks, "return_lse": True}
    if max(news) > 1:
        given.update(starts=starts, max_new=max(news))
    results = [cache.attend(q, **given)]
    if shift:
        results.append(cache.attend(off_by_one(q), **given))
    if news == lengths:
        k, v = (torch.cat([x[i][0] for x in seqs]).to(DEV) for i in (0, 1))
        results.append(window_attention(ctx, q, *((off_by_one(x) if shift else x) for x in (k, v)),
                                        starts=starts, max_length=max(news), window=window,
                                        sinks=sinks, return_lse=True))
    for i, (kk, vv) in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        o, l, t = attended_at_once(q[a:b], kk[0], vv[0], d ** -0.5, window, sinks)
        for out, lse in results:
            check(out[a:b], o, t)
            check_norm(out[a:b], o, dtype)
            check(lse[a:b], l, 2.0 ** -16 * (1 + l.abs()))


def test_slots_known_on_the_host(ctx):
    """A slot twice would lose the pages taken for it first, one that is not
    there would grow nothing: refused where the host knows, like a fork's."""
    from vectorstorekit_amd import VSKError

    cache, _ = filled(ctx, [20, 4], 16, 2, 64, F32, poison=False)
    table, refs = cache.table.clone(), cache.refs.clone()
    for f, *a in ((cache.reserve, [0, 0], [16, 16]), (cache.reserve, np.array([1, 2]), [1, 1]),
                  (cache.reserve, [-1], [1]), (cache.free, [2]), (cache.free, [-1]),
                  (cache.fork, [0], [2]), (cache.fork, [0, 0], [1, 1])):
        with pytest.raises(VSKError) as e:
            f(*a)
        assert e.value.kind == "invalidArgument"
    assert torch.equal(cache.table, table) and torch.equal(cache.refs, refs)
    assert cache.lengths.tolist() == [20, 4]
    cache.reserve([], [])
    cache.free([])
    cache.reserve((1, 0), np.array([1, 2]))
    assert cache.lengths.tolist() == [22, 5]
    cache.fork([0], np.array([1]))
    cache.free(ints([1, 1, 7]))  # (on the GPU: slots out of range hold nothing)
    assert cache.lengths.tolist() == [22, 0]


def test_layers_past_32_bits(ctx):
    from vectorstorekit_amd import VSKError

    cache, _ = filled(ctx, [20, 4], 16, 2, 64, F32, poison=False)
    k, x = cache.k.clone(), torch.ones(2, 2, 64, device=DEV)
    for layer in (1, -1, 1 << 32, -(1 << 32)):  # (not layer 0)
        for f in (lambda: cache.append(x, x, layer=layer), lambda: cache.attend(x, layer=layer)):
            with pytest.raises(VSKError) as e:
                f()
            assert e.value.kind == "invalidArgument"
    assert torch.equal(cache.k, k)


def test_page_keeping_beyond_its_counts(ctx):
    """More pages or slots than the kernels count are refused, not launched."""
    import ctypes

    cache, _ = filled(ctx, [20, 4], 16, 2, 64, F32, poison=False)
    for field in ("pages", "slots"):
        kv = type(cache._kv).from_buffer_copy(cache._kv)
        setattr(kv, field, (1 << 30) + 1)
        assert ctx.lib.vsk_kv_compact(ctx.handle, None, ctypes.byref(kv)) == -9


def test_refusals(ctx):
    from vectorstorekit_amd import PagedKVCache, RotaryEmbedding, VSKError, window_attention

    def refused(kind, f, *a, **k):
        with pytest.raises(VSKError) as e:
            f(*a, **k)
        assert e.value.kind == kind, e.value

    bad = "invalidArgument"
    for args in ({"layout": "spiral"}, {"rotary_dim": 7}, {"rotary_dim": 80}, {"base": 0.0},
                 {"scaling": {"type": "linear"}}, {"scaling": {"type": "who", "factor": 2}},
                 {"scaling": {"type": "yarn", "factor": 2}},
                 {"scaling": {"type": "ntk", "factor": 2, "more": 1}}):
        refused(bad, RotaryEmbedding, ctx, 64, **args)
    rope = RotaryEmbedding(ctx, 64)
    x = torch.zeros(3, 2, 64, device=DEV)
    pos = ints([0, 1, 2])
    refused("dimensionMismatch", rope.apply, x[..., :32], positions=pos)
    refused("dimensionMismatch", rope.apply, x, positions=pos[:2])
    refused(bad, rope.apply, x, positions=pos.long())
    refused(bad, rope.apply, x.cpu(), positions=pos)
    refused("unsupportedOperation", rope.apply, x.double(), positions=pos)
    assert rope.apply(x[:0], positions=pos[:0]).shape == (0, 2, 64)

    cache, _ = filled(ctx, [20, 4], 16, 2, 64, F32, poison=False)
    k, v, t, n = cache.k, cache.v, cache.table, cache.lengths
    refused("unsupportedOperation", PagedKVCache.over, ctx, k[:, :, :8], v[:, :, :8], t, n)
    refused("dimensionMismatch", PagedKVCache.over, ctx, k, v[:, :, :, :1], t, n)
    refused("dimensionMismatch", PagedKVCache.over, ctx, k, v, t, n[:1])
    refused(bad, PagedKVCache.over, ctx, k, v, t.long(), n)
    refused("unsupportedOperation", PagedKVCache.over(ctx, k, v, t, n).compact)
    refused("unsupportedOperation", PagedKVCache, ctx, pages=4, page_size=24, kv_heads=1,
            head_dim=8, slots=1, width=1)
    q = torch.zeros(2, 4, 64, device=DEV)
    refused("dimensionMismatch", cache.attend, q[:, :3])
    refused("dimensionMismatch", cache.attend, q[..., :32])
    refused(bad, cache.attend, q.half())
    refused(bad, cache.attend, torch.zeros(3, 4, 64, device=DEV))  # more than the slots
    refused(bad, cache.attend, q, scale=0.0)
    refused(bad, cache.attend, q, scale=math.inf)
    refused(bad, cache.attend, q, window=0)
    refused(bad, cache.attend, q, sinks=-1)
    refused(bad, cache.attend, q, layer=1)
    refused("dimensionMismatch", cache.attend, q, seqs=[0])
    refused("dimensionMismatch", cache.append, x[:2], x[:2, :1])
    refused("dimensionMismatch", cache.append, x[:2], x[:1])
    refused("dimensionMismatch", cache.append, x[:2], x[:2], rotary=RotaryEmbedding(ctx, 32))
    refused(bad, cache.fork, [0], [0])
    refused(bad, cache.fork, [0, 0], [1, 1])
    refused(bad, cache.fork, [0], [2])
    refused("dimensionMismatch", cache.reserve, [0, 1], [1])
    refused("dimensionMismatch", window_attention, ctx, x, x[:, :, :32], x, starts=[0, 3])
    refused("dimensionMismatch", window_attention, ctx, x, x[:2], x[:2], starts=[0, 3])
    refused("dimensionMismatch", window_attention, ctx, x, x, x, starts=[0, 3], k_starts=[0])
    refused(bad, window_attention, ctx, x, x.half(), x, starts=[0, 3])
    big = torch.zeros(1, 1, 320, device=DEV)
    refused("unsupportedOperation", window_attention, ctx, big, big, big, starts=[0, 1])
    # more keys than positions hold (one row, seen very often)
    far = torch.zeros(1, 1, 8, device=DEV).expand((1 << 30) + 1, 1, 8)
    refused("invalidBufferSize", window_attention, ctx, x[..., :8], far, far, starts=[0, 3],
            k_starts=[0, 3])
    far = torch.zeros(1, 16, 1, 8, device=DEV).expand(1 << 31, 16, 1, 8)
    refused("invalidBufferSize", PagedKVCache.over, ctx, far, far, t, n)
    assert cache.attend(q[:0]).shape == (0, 4, 64)
    # nothing was lost on the way
    assert int(cache.lengths[0]) == 20 and cache.missing() == 0
