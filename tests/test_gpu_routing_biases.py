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
