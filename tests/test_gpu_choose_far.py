"""The choice's order where scores no longer tell experts apart, or are about to leave the range of 64 bits."""
import math

import pytest
import torch

from test_gpu_choose import plain_many

pytestmark = pytest.mark.gpu


def in_groups(T, dtype, seed, ranges, size=8):
    """T tokens of len(ranges) groups: a group's first two logits at `first`, the others whole numbers of `rest`, shuffled."""
    g = torch.Generator().manual_seed(seed)
    parts = []
    for first, (low, high) in ranges:
        part = torch.randint(low, high + 1, (T, size), generator=g).float()
        if first is not None:
            part[:, :2] = first + torch.rand(T, 2, generator=g)
        parts.append(part.gather(1, torch.rand(T, size, generator=g).argsort(1)))
    return torch.cat(parts, 1).to(dtype).cuda()


# what the groups hold: the second and the last are ahead by far, so which two are kept is plain
SATURATED = [(None, (-4, -2)), (None, (30, 100)), (None, (-4, -2)), (None, (33, 90))]
VERY_LOW = [(None, (-60, -40)), (2.0, (-3000, -701)), (None, (-60, -40)), (2.0, (-3000, -701))]
FAR_BELOW = [(None, (-90, -60)), (5.0, (-3000, -701)), (None, (-90, -60)), (5.0, (-3000, -701))]


@pytest.mark.parametrize("T", [1, 50, (1 << 14) + 77])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring,ranges", [("sigmoid", SATURATED), ("sigmoid", VERY_LOW), ("softmax", FAR_BELOW)])
def test_order_is_the_logits_in_groups_by_sums(backend, gpu, scoring, ranges, dtype, T):
    """Without a bias the experts of the kept groups come in the logits' order, however the groups are ranked; equal
    logits by index."""
    l = in_groups(T, dtype, 3, ranges)
    how = dict(scoring=scoring, num_groups=4, top_groups=2, group_score="sum2")
    want = plain_many(l, 12, None, scoring, 4, 2, "sum2")
    assert bool(((want // 8) % 2 == 1).all())                          # of the second and the last group
    ids, w = backend.choose_experts(l, 12, **how)
    assert torch.equal(ids, want)
    assert torch.equal(ids, backend.choose_experts(l, 12, **{**how, "group_score": "max"})[0])
    picked = l.gather(1, ids.long()).double()
    assert bool((picked[:, 1:] <= picked[:, :-1]).all()) and bool((w[:, 1:] <= w[:, :-1]).all())


def test_unavailable_experts_stay_so_in_groups_by_sums(backend, gpu):
    """-inf, and a NaN ahead of all, as with groups by their greatest."""
    l = in_groups(40, torch.float32, 5, SATURATED)
    l[:, 9::3] = -math.inf
    l[5:10, 8] = math.nan
    l[10:15, 31] = math.inf
    l[15] = -math.inf
    how = dict(scoring="sigmoid", num_groups=4, top_groups=2)
    ids, _ = backend.choose_experts(l, 12, group_score="sum2", **how)
    assert torch.equal(ids, backend.choose_experts(l, 12, group_score="max", **how)[0])
    assert bool((ids[5:10, 0] == 8).all()) and bool((ids[15] == -1).all()) and bool((ids[:, 11] == -1).any())


@pytest.mark.parametrize("T", [1, 60, (1 << 13) + 77])
@pytest.mark.parametrize("E,groups,top", [(64, 1, 1), (64, 8, 3), (20, 5, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_down_to_the_end_of_the_range(backend, gpu, monkeypatch, scoring, E, groups, top, T):
    """With a bias of zeros the order is the scores', as far as 64 bits hold them: logits of whole numbers down to -730,
    whose scores (2^-1053) lie a factor e apart, well above the 2^-1064 that the keys keep; at -800 and below a score is 0,
    and still available."""
    g = torch.Generator().manual_seed(E + T)
    l = -torch.rand(T, E, generator=g).argsort(1).float() - (731 - E)            # whole numbers, each once
    top_one = -800.0 if scoring == "sigmoid" else 0.0                             # softmax: what the others are far below
    l[:, 0] = top_one
    if T > 1:
        l[1::4, 5:9] = -math.inf
        l[2::4, 9:12] = -1000.0
    l = l.cuda()
    # torch's own is 0 below -709.8, where its exp(-l) leaves the range; exp(l) is within a factor 1 + exp(-667) of it
    monkeypatch.setattr(torch, "sigmoid", torch.exp)
    zeros, k = torch.zeros(E, device="cuda"), E // groups * top
    for group_score in ("max", "sum2"):
        ids, _ = backend.choose_experts(l, k, zeros, scoring=scoring, num_groups=groups, top_groups=top, group_score=group_score)
        want = plain_many(l, k, zeros, scoring, groups, top, group_score)
        assert torch.equal(ids, want)
    if groups == 1:
        there = ids >= 0
        picked = torch.where(there, l.gather(1, ids.clamp(min=0).long()), -math.inf)
        low = picked < -745.2                                                     # scores of 0: by index
        assert bool(((picked[:, 1:] <= picked[:, :-1]) | low[:, :-1]).all())
