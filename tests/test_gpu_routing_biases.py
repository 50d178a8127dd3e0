"""The choice of experts under biases far from the scores: infinite ones, and large ones of both signs, against the definition in 64 bits."""

import math

import pytest
import torch

import int8_reference as ref
import llmoop_b200 as nb
from test_gpu_int8 import _route_reference

pytestmark = pytest.mark.gpu

GROUPS = [dict(groups=1), dict(experts=64, groups=8, chosen_groups=3), dict(experts=256, groups=8, chosen_groups=4, group_scores=2), dict(experts=96, groups=3, chosen_groups=2),
          dict(experts=244, groups=4, chosen_groups=2, group_scores=2), dict(experts=244, groups=4, chosen_groups=1)]  # the last two: groups that are no runs of threads


def agrees(logits, bias, r):
    ids, weights = ref.route(logits, bias, r)
    want_ids, want = _route_reference(logits, bias, r)
    assert torch.equal(ids, want_ids)
    # one rounding of the weight, 2^-40 for exponentials and sums in 64 bits
    assert bool(((weights.double() - want).abs() <= want.abs() * (ref.F32 + 2.0 ** -40) + 1e-44).all())


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("top_k", [1, 2, 8, 40])
@pytest.mark.parametrize("groups", GROUPS, ids=lambda how: f"{how.get('experts', 128)}g{how['groups']}")
def test_infinite_biases(groups, top_k, sigmoid):
    """An expert with a bias of +inf comes before all others, several of them by their numbers, closed ones not at all."""
    how = {"experts": 128, "chosen_groups": 1} | groups
    r = nb.Routing(**how, top_k=min(top_k, how["experts"] // how["groups"] * how["chosen_groups"]), sigmoid=sigmoid)
    g = ref.generator(r.experts + top_k)
    logits = torch.randn((24, r.experts), generator=g, device="cuda") * 2
    logits[8:16].masked_fill_(torch.rand((8, r.experts), generator=g, device="cuda") < 0.5, -math.inf)
    logits[23] = -math.inf
    for hot in ([r.experts - 3], [5, 7], [r.experts // 2, 3, r.experts - 1, 4], range(0, r.experts, 3), range(r.experts)):
        bias = torch.randn(r.experts, generator=g, device="cuda") * 0.1
        bias[list(hot)] = math.inf
        bias[[1, r.experts // 3]] = torch.tensor([-math.inf, math.nan], device="cuda")
        for kind in (torch.float32, torch.bfloat16):
            agrees(logits.to(kind), bias, r)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("large", [3e2, 1e4, 1e6, 1e9, 1e15, 1e32])
@pytest.mark.parametrize("how", [dict(experts=16, top_k=2, groups=8, chosen_groups=3), dict(experts=64, top_k=4, groups=32, chosen_groups=9), dict(experts=256, top_k=6, groups=8, chosen_groups=4),
                                 dict(experts=70, top_k=3, groups=7, chosen_groups=2), dict(experts=244, top_k=2, groups=4, chosen_groups=1), dict(experts=1022, top_k=3, groups=2, chosen_groups=1)],
                         ids=lambda how: f"{how['experts']}g{how['groups']}")
def test_groups_of_large_biases_of_both_signs(how, large, sigmoid):
    """A group's two largest choices cancel, and what is left of its rank is smaller than what 32 bits lose of either."""
    r, size = nb.Routing(**how, sigmoid=sigmoid, group_scores=2), how["experts"] // how["groups"]
    g = ref.generator(r.experts)
    logits = torch.randn((64, r.experts), generator=g, device="cuda") * torch.logspace(-5, 0.5, 64, device="cuda")[:, None]
    for normal in (0, 1, r.groups):  # groups whose biases are small
        for open_ in (2, size):
            bias = torch.full((r.groups, size), -large, device="cuda")
            first = torch.rand((r.groups, size), generator=g, device="cuda").argsort(dim=1)
            bias.scatter_(1, first[:, :1], large)
            bias[:normal] = 0.0
            bias.scatter_(1, first[:, open_:], -math.inf)
            agrees(logits, bias.flatten(), r)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("lowest", [-1e9, float(torch.finfo(torch.float32).min), float(torch.finfo(torch.bfloat16).min)])
@pytest.mark.parametrize("group_scores", [1, 2])
@pytest.mark.parametrize("count,groups,chosen", [(128, 1, 1), (256, 8, 4), (64, 32, 5), (244, 4, 2)])
def test_biases_of_the_lowest_value(count, groups, chosen, group_scores, lowest, sigmoid):
    """A mask by finite biases: experts, all but one of a group, whole groups, all groups but one, all."""
    r, size = nb.Routing(experts=count, top_k=min(6, count // groups * chosen), sigmoid=sigmoid, groups=groups, chosen_groups=chosen, group_scores=group_scores), count // groups
    g = ref.generator(count)
    logits = torch.randn((16, count), generator=g, device="cuda") * 2
    for masked in (torch.rand(count, generator=g, device="cuda") < 0.5, torch.arange(count, device="cuda") % size > 0, torch.arange(count, device="cuda") // size < groups // 2,
                   torch.arange(count, device="cuda") // size != groups - 1, torch.ones(count, dtype=torch.bool, device="cuda")):
        agrees(logits, (torch.randn(count, generator=g, device="cuda") * 0.1).masked_fill(masked, lowest), r)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("count,groups,chosen", [(40, 8, 3), (256, 8, 4), (64, 32, 9), (244, 4, 2)])
def test_closed_groups_beside_groups_of_the_lowest_biases(count, groups, chosen, sigmoid):
    """Two choices of the lowest value add up to -infinity in 32 bits; the group stays in front of those without an open expert."""
    r, size = nb.Routing(experts=count, top_k=min(8, count // groups * chosen), sigmoid=sigmoid, groups=groups, chosen_groups=chosen, group_scores=2), count // groups
    g = ref.generator(count)
    lowest = float(torch.finfo(torch.float32).min)
    logits = torch.randn((groups + 8, count), generator=g, device="cuda")
    closed = torch.rand((groups + 8, groups), generator=g, device="cuda") < 0.7
    closed[:groups] = torch.ones((groups, groups), dtype=torch.bool, device="cuda") ^ torch.eye(groups, dtype=torch.bool, device="cuda")  # one group is open, each in turn
    logits.masked_fill_(closed.repeat_interleave(size, dim=1), -math.inf)
    for masked in (torch.ones(count, dtype=torch.bool, device="cuda"), torch.rand(count, generator=g, device="cuda") < 0.8, torch.arange(count, device="cuda") // size != groups - 1):
        agrees(logits, (torch.randn(count, generator=g, device="cuda") * 0.1).masked_fill(masked, lowest), r)


@pytest.mark.parametrize("apart", [1e-9, 1e-11])
@pytest.mark.parametrize("middle", [0.0, 12.0, 19.0])
def test_candidates_that_a_bias_of_a_billionth_tells_apart(apart, middle):
    """Scores equal or next to one another in 32 bits, and choices that 64 bits hold apart by more than their exponentials' error."""
    g = ref.generator(5)
    logits = middle + torch.randint(0, 3, (64, 128), generator=g, device="cuda") * 2.0 ** -18
    bias = torch.randn(128, generator=g, device="cuda") * apart
    for some in (bias, bias + 0.25):
        agrees(logits, some, nb.Routing(experts=128, top_k=8, sigmoid=True))
