"""Calls of ``share`` and ``attend(shared=)`` that their documents allow or
refuse, past those of test_gpu_shared.py (whose tolerances these are)."""
import pytest
import torch

from test_gpu_shared import BF, cache_of, check_shared, gen, ints, normal, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("host", [True, False])
def test_fewer_sequences_than_the_plan(ctx, host):
    """A plan with slots of its own serves its first sequences, a group cut
    through among them."""
    from vectorstorekit_amd import VSKError

    g = gen(1)
    cache, slots = cache_of(ctx, g, [(64, [3, 40, 5, 6]), (96, [10, 20])], 32, 2, 64, BF,
                            order=[4, 0, 5, 2, 1, 3])
    plan = cache.share([0, 4, 6], seqs=slots if host else ints(slots))
    assert plan.prefix.tolist() == [64] * 4 + [96] * 2
    for n in (6, 5, 4, 2, 1):
        q = normal(g, n, 4, 64, dtype=BF)
        check_shared(cache, slots, q, None, cache.attend(q, shared=plan), 0.125)
        at = starts_of([i % 3 for i in range(n)])
        q = normal(g, at[-1], 4, 64, dtype=BF)
        for starts in (at, ints(at)):
            out = cache.attend(q, shared=plan, starts=starts, max_new=2)
            check_shared(cache, slots, q, at, out, 0.125)
    assert cache.attend(q[:0], shared=plan).shape == (0, 4, 64)
    assert cache.attend(q[:0], shared=plan, starts=[0]).shape == (0, 4, 64)
    for starts in ([], [0] * 8, ints([0] * 8)):
        with pytest.raises(VSKError):
            cache.attend(q, shared=plan, starts=starts)


def test_descending_groups_of_unsigned_numbers(ctx):
    """They descend whatever their type, whose differences wrap around."""
    import numpy as np

    from vectorstorekit_amd import VSKError

    cache, _ = cache_of(ctx, gen(2), [(32, [3, 4, 5])], 32, 2, 64, BF)
    for dtype in (np.uint8, np.uint32, np.uint64, np.int64):
        assert cache.share(np.array([0, 1, 3], dtype)).prefix.tolist() == [32, 32, 32, 0]
        with pytest.raises(VSKError):
            cache.share(np.array([0, 3, 1], dtype))
