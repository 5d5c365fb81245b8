"""``ops.topk_routing`` with groups that hold NaN: a NaN score comes last, and so does a group whose score is NaN; never more than ``group_topk``
groups take part."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rank(values):
    """Indices best first: NaN last, ties to the lower index."""
    return sorted(range(len(values)), key=lambda i: (values[i] != values[i], 0.0 if values[i] != values[i] else -values[i], i))


def _choice(scores, groups, group_topk, topk):
    per = len(scores) // groups
    take = max(1, min(topk // group_topk, per))
    sums = []
    for g in range(groups):
        mine = scores[g * per:(g + 1) * per]
        total = 0.0
        for i in _rank(mine)[:take]:
            total += mine[i]
        sums.append(total)
    kept = set(_rank(sums)[:group_topk])
    alive = [e for e in range(len(scores)) if e // per in kept]
    return [alive[i] for i in _rank([scores[e] for e in alive])[:topk]]


@pytest.mark.parametrize("experts,groups,group_topk,topk", [(8, 4, 1, 2), (24, 6, 2, 4), (24, 6, 3, 3), (60, 5, 2, 8), (256, 8, 4, 8), (128, 64, 7, 14)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_groups_that_hold_nan(gpu, experts, groups, group_topk, topk, score, with_bias):
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(experts + topk)
    rows = 60
    logits = torch.randn(rows, experts, generator=gen)
    share = torch.tensor([0.0, 0.05, 0.3, 0.6, 0.9, 1.0]).repeat(rows // 6)[:, None]
    logits[torch.rand(rows, experts, generator=gen) < share] = math.nan
    bias = torch.randn(experts, generator=gen) * 0.1 if with_bias else torch.zeros(experts)
    scores = ((torch.sigmoid(logits.double()) if score == "sigmoid" else torch.softmax(logits.double(), 1)) + bias.double()).tolist()
    _, idx, _ = ops.topk_routing(logits.to(gpu), topk, score_function=score, expert_bias=bias.to(gpu) if with_bias else None, num_groups=groups, group_topk=group_topk)
    for t, row in enumerate(idx.tolist()):
        assert row == _choice(scores[t], groups, group_topk, topk), t
