"""``ops.topk_routing`` with groups whose biased scores are large and of both signs: their sum is small, and what fp32 loses in it goes by
the terms.  The indices are those of the sums in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size", [50.0, 400.0])
def test_terms_that_cancel(gpu, score, size):
    """Two experts of every group have opposite biases, each group its own, so that experts lie far apart; the groups' sums differ by a few
    steps of an fp32 number of the biases' size."""
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(int(size))
    rows, groups, per, group_topk, topk = 500, 8, 4, 2, 4
    bias = torch.full((groups, per), -4.0 * size)
    bias[:, 1] = size * (1.0 + 0.3 * torch.arange(groups))
    bias[:, 2] = -bias[:, 1]
    bias = bias.reshape(-1)
    logits = (torch.rand(rows, 1, 1, generator=gen) - 0.5) + torch.randint(-8, 9, (rows, groups, 1), generator=gen) * (size * 2.0 ** (-24 if score == "sigmoid" else -20)) + torch.rand(rows, groups, per, generator=gen) * 2.0 ** -22
    logits = logits.reshape(rows, -1)
    order = (torch.sigmoid(logits.double()) if score == "sigmoid" else torch.softmax(logits.double(), 1)) + bias.double()
    g = order.view(rows, groups, per)
    best = torch.sort(g, dim=2, descending=True).values[:, :, :2].sum(2)
    ranked = torch.sort(best, dim=1, descending=True)
    clear = ranked.values[:, group_topk - 1] - ranked.values[:, group_topk] > size * 2.0 ** -48       # 64 bits tell them apart
    kept = torch.zeros(rows, groups, dtype=torch.bool).scatter(1, ranked.indices[:, :group_topk], True)
    want = torch.where(kept[:, :, None], g, -torch.inf).reshape(rows, -1).topk(topk, dim=1).indices
    assert int(clear.sum()) > rows // 2
    _, idx, _ = ops.topk_routing(logits.to(gpu), topk, score_function=score, expert_bias=bias.to(gpu), num_groups=groups, group_topk=group_topk)
    wrong = (idx.cpu() != want).any(1) & clear
    assert not bool(wrong.any()), (int(wrong.sum()), int(clear.sum()))


def test_scores_below_the_smallest_normal_number(gpu):
    """One expert has all of the softmax but 2^-28: of the other groups, one with an expert above and one below 2^-126 beats one with
    both just above."""
    from primus_amd.pytorch import ops

    row = torch.tensor([0.0, -20.0, -87.300, -87.340, -87.325, -87.325, -95.0, -95.0])
    p = torch.softmax(row.double(), 0)
    assert p[3] < 2.0 ** -126 < p[5] < p[2] and float(p[2] + p[3]) > 1.004 * float(p[4] + p[5])
    _, idx, _ = ops.topk_routing(row[None].repeat(3, 1).to(gpu), 4, num_groups=4, group_topk=2)
    assert idx.tolist() == [[0, 1, 2, 3]] * 3
