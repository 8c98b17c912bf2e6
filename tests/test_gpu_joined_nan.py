"""A query or a key that is NaN gives its row NaN also where the row's keys were
divided into parts (cross attention over long sets, shared prefixes): exactly
the rows that it gives NaN in the plain attention, and no others."""
import math

import pytest
import torch

from test_gpu_kvcache import kernels_of
from test_gpu_shared import BF, F16, F32, cache_of, gen, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("new,heads,kv,d", [(1, 8, 8, 64), (6, 4, 1, 64), (3, 4, 2, 100),
                                            (2, 8, 1, 256), (300, 8, 1, 128)])
def test_cross_parts(ctx, dtype, new, heads, kv, d):
    from vectorstorekit_amd import cross_attention

    g = gen(new)
    length = 20001
    q = normal(g, new, heads, d, dtype=dtype)
    k, v = (normal(g, length, kv, d, dtype=dtype) for _ in range(2))
    row, head = new // 2, heads - 1
    q[row, head, d // 2] = math.nan
    (out, lse), used = kernels_of(ctx, lambda: cross_attention(
        ctx, q, k, v, starts=[0, new], k_starts=[0, length], return_lse=True))
    assert "attn_join" in used
    bad = torch.zeros(new, heads, dtype=torch.bool)
    bad[row, head] = True
    assert torch.equal(torch.isnan(lse).cpu(), bad)
    assert torch.equal(torch.isnan(out).all(-1).cpu(), bad)
    assert bool(torch.isfinite(out[~bad]).all()) and bool(torch.isfinite(lse[~bad]).all())


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 64), (5, 5, 80), (8, 1, 256), (3, 1, 37)])
def test_shared(ctx, dtype, heads, kv, d):
    """A query of one branch; then all shared keys, of which a whole part is NaN."""
    g = gen(d)
    cache, slots = cache_of(ctx, g, [(512, [40, 3, 17, 100]), (64, [20, 5])], 32, kv, d, dtype)
    plan = cache.share([0, 4, 6])
    q = normal(g, 6, heads, d, dtype=dtype)
    q[2, heads // 2, 0] = math.nan
    bad = torch.zeros(6, heads, dtype=torch.bool)
    bad[2, heads // 2] = True
    out, lse = cache.attend(q, shared=plan, return_lse=True)
    assert torch.equal(torch.isnan(out).all(-1).cpu(), bad)
    assert torch.equal(torch.isnan(lse).cpu(), bad)
    assert bool(torch.isfinite(out[~bad]).all()) and bool(torch.isfinite(lse[~bad]).all())
    cache.k[cache.table[0, :16].long()] = math.nan
    out, lse = cache.attend(q, shared=plan, return_lse=True)
    bad[:4] = True
    assert torch.equal(torch.isnan(out).all(-1).cpu(), bad)
    assert torch.equal(torch.isnan(lse).cpu(), bad)
    assert bool(torch.isfinite(out[~bad]).all()) and bool(torch.isfinite(lse[~bad]).all())
