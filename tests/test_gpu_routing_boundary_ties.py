"""``ops.topk_routing`` where the last expert chosen and the first left out have the same logit and the same bias, and an expert behind them
is nearer to the two than fp32 scores tell: the indices are those of the scores in 64 bits, equal index for index."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _better(order):
    e = torch.arange(order.shape[1])
    return ((order[:, None, :] > order[:, :, None]) | ((order[:, None, :] == order[:, :, None]) & (e[None, :] < e[:, None]))).sum(2)


def _choice(logits, bias, topk, score, groups=1, group_topk=1):
    l = logits.double().cpu()
    order = (torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, 1)) + bias.double().cpu()
    if groups > 1:
        t, e = order.shape
        g = order.view(t, groups, e // groups)
        take = max(1, min(topk // group_topk, e // groups))
        best = torch.sort(g, dim=2, descending=True).values[:, :, :take].sum(2)
        order = torch.where((_better(best) < group_topk)[:, :, None], g, -torch.inf).reshape(t, e)
    place = _better(order)
    return torch.stack([(place == k).to(torch.int8).argmax(1) for k in range(topk)], 1)


def _check(gpu, logits, bias, topk, score, groups=1, group_topk=1):
    from primus_amd.pytorch import ops

    probs, idx, counts = ops.topk_routing(logits.to(gpu), topk, score_function=score, expert_bias=bias.to(gpu), num_groups=groups if groups > 1 else None,
                                          group_topk=group_topk if groups > 1 else None)
    want = _choice(logits, bias, topk, score, groups, group_topk)
    wrong = (idx.cpu() != want).any(1).nonzero().reshape(-1)
    assert wrong.numel() == 0, (wrong.numel(), logits[wrong[0]].tolist(), idx[wrong[0]].tolist(), want[wrong[0]].tolist())
    assert torch.equal(counts.cpu(), torch.bincount(want.reshape(-1), minlength=logits.shape[1]))


@pytest.mark.parametrize("score,row,bias,topk,want", [("sigmoid", [20.0, 20.0, 25.0], 0.0, 1, [2]), ("softmax", [0.0, -25.0, -25.0, -24.5], 0.05, 2, [0, 3])])
def test_a_better_expert_behind_a_tie(gpu, score, row, bias, topk, want):
    logits, b = torch.tensor([row]), torch.full((len(row),), bias)
    assert _choice(logits, b, topk, score).tolist() == [want]
    _check(gpu, logits, b, topk, score)


def test_a_better_sum_behind_a_tie(gpu):
    """Two experts of 0.5 exactly and one whose score and bias add up to 0.5 but for what an fp32 sum loses."""
    gen = torch.Generator().manual_seed(1)
    better = 0
    for x in (torch.rand(60, generator=gen) * 4 - 2).tolist():
        logits = torch.tensor([[0.0, 0.0, x]])
        bias = torch.tensor([0.0, 0.0, float(0.5 - torch.sigmoid(logits[0, 2].double()))])
        better += int(_choice(logits, bias, 1, "sigmoid")[0, 0] == 2)
        _check(gpu, logits, bias, 1, "sigmoid")
    assert 10 < better < 50


@pytest.mark.parametrize("experts,groups,group_topk", [(3, 1, 1), (8, 1, 1), (8, 4, 3), (60, 1, 1), (64, 8, 3), (256, 1, 1), (256, 8, 4), (1023, 33, 20), (1024, 1, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [0.0, 0.0625])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_few_values_whose_scores_fp32_cannot_tell(gpu, experts, groups, group_topk, score, bias, dtype):
    """Logits of few values far out, as bf16 logits and equal biases give them: rows full of ties, at the boundary too."""
    gen = torch.Generator().manual_seed(experts + groups)
    rows = 40 if experts > 256 else 300
    values = torch.randint(0, 9, (rows, experts), generator=gen).float()
    if score == "sigmoid":
        logits = 16.0 + values
    else:
        logits = -20.0 - values
        logits[torch.arange(rows), torch.randint(0, experts, (rows,), generator=gen)] = 0.0
    logits[0] = 0.0
    logits[1] = logits[1, 0]
    for topk in (1, 2, 6, 8):
        if topk < experts and topk <= group_topk * (experts // groups):
            _check(gpu, logits.to(dtype), torch.full((experts,), bias), topk, score, groups, group_topk)
