"""Shared prefixes of sequences that are cut back (their lengths lowered to
whole pages) and grow again: ``reserve`` gives them pages of their own in place
of shared ones, and the plan is made anew.  Tolerances: test_gpu_shared.py."""
import pytest
import torch

from test_gpu_shared import BF, F32, check_shared, forked, ints, normal, view

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cut,left", [([1], 64), ([4], 0), ([2], 176), ([1, 5], 96), ([3], 192)])
@pytest.mark.parametrize("grown", [1, 20, 120])
def test_cut_back_and_grown_again(ctx, dtype, cut, left, grown):
    """The first member, others, several; to nothing, to the last shared page,
    to the prefix's end; growing by a token, within the old prefix and past it."""
    cache, slots, g = forked(ctx, dtype)
    plan = cache.share([0, 5], seqs=slots)
    assert plan.prefix.tolist() == [192] * 5
    for slot in cut:
        cache.lengths[slot] = left
    q = normal(g, 5, 8, 64, dtype=dtype)
    if left:  # (cut back alone: what was found holds)
        one, order = view(cache, slots)
        check_shared(one, order, q, None, cache.attend(q, shared=plan), 0.125)
    cache.reserve(cut, [grown] * len(cut))
    assert cache.missing() == 0
    new = [grown * i for i in range(len(cut) + 1)]
    cache.append(*(normal(g, new[-1], 2, 64, dtype=dtype) for _ in range(2)), starts=new, seqs=cut)
    plan.update()
    # pages of their own from the cut on, of which none is shared
    assert plan.prefix.tolist() == [min(left, 192)] * 5
    one, order = view(cache, slots)
    check_shared(one, order, q, None, cache.attend(q, shared=plan), 0.125)
    # the others still share all that they did
    rest = [s for s in range(1, 6) if s not in cut]
    plan = cache.share(ints([0, len(rest)]), seqs=rest)
    assert plan.prefix.tolist() == [192] * len(rest)
    one, _ = view(cache, slots)
    check_shared(one, rest, q[:len(rest)], None, cache.attend(q[:len(rest)], shared=plan), 0.125)


@pytest.mark.parametrize("left", [0, 64, 100, 176, 192, 195])
@pytest.mark.parametrize("grown", [1, 40, 110])
def test_pages_written_over_are_given_back(ctx, left, grown):
    """A page's count is that of the table entries that name it, also of those
    that new pages took the place of; freed, none is left."""
    cache, slots, _ = forked(ctx)

    def counted():
        held = cache.table[cache.table >= 0].long()
        assert torch.equal(torch.bincount(held, minlength=cache.pages).int(), cache.refs)

    counted()
    for _ in range(6):  # (64 pages would not last)
        for slot in (1, 3):
            cache.lengths[slot] = left
        cache.reserve([1, 3], [grown, 1])
        assert cache.missing() == 0
        assert cache.lengths[[1, 3]].tolist() == [left + grown, left + 1]
        counted()
    cache.compact()
    counted()
    cache.free(range(7))
    assert not cache.refs.any() and bool((cache.table == -1).all())
