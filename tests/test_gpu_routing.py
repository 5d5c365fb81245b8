"""``ops.topk_routing`` against its definition in 64 bits: the choice of experts (equal index for index, ties and scores nearer to
each other than fp32 can tell included), probabilities, counts and the logits' gradient.

Tolerances.  A score's relative error is at most (x + 40) 2^-24 (x = distance to the row's largest logit, below 40 here: the
rounding of x, expf, at most 38 additions and a quotient); a renormalised one has it twice: below 2^-17.  A gradient is a
product of three such numbers and of a difference whose terms have them too: 2^-15 of the sum of the terms' magnitudes, plus
half a step of the logits' type (and of its smallest number, where the value underflows)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _better(order):
    """place[t, e]: how many experts are ahead of e; ties to the lower index."""
    e = torch.arange(order.shape[1])
    ahead = (order[:, None, :] > order[:, :, None]) | ((order[:, None, :] == order[:, :, None]) & (e[None, :] < e[:, None]))
    return ahead.sum(2)


def _reference(logits, topk, score="softmax", bias=None, groups=1, group_topk=1, renorm=True, scale=1.0, mask=None, dprobs=None):
    l = logits.double().cpu()
    t, e = l.shape
    p = torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, 1)
    order = l if bias is None and groups == 1 else p if bias is None else p + bias.double().cpu()
    if groups > 1:
        g = order.view(t, groups, e // groups)
        take = max(1, min(topk // group_topk, e // groups))
        best = torch.sort(g, dim=2, descending=True).values[:, :, :take].sum(2)
        order = torch.where((_better(best) < group_topk)[:, :, None], g, -math.inf).reshape(t, e)
    place = _better(order)
    idx = torch.stack([(place == k).to(torch.int8).argmax(1) for k in range(topk)], 1)
    w = p.gather(1, idx)
    total = w.sum(1, keepdim=True) + (1e-20 if score == "sigmoid" else 0.0)
    share = w / total if renorm else w
    if renorm and score == "softmax":           # of the chosen logits; 0 where all of them are -inf
        share = torch.softmax(l.gather(1, idx), 1)
        share = torch.where((l.gather(1, idx) == -math.inf).all(1, keepdim=True), 0.0, share)
    probs = share * scale
    live = torch.ones(t, 1, dtype=torch.bool) if mask is None else mask.cpu().bool()[:, None]
    out = {"probs": torch.where(live, probs, 0.0), "indices": torch.where(live, idx, -1)}
    out["counts"] = torch.bincount(out["indices"][out["indices"] >= 0], minlength=e)
    if dprobs is not None:
        g = dprobs.double().cpu() * scale
        ga = g.abs()
        zeros = torch.zeros_like(p)
        if renorm:
            g, ga = (g - (g * share).sum(1, keepdim=True)) / total, (ga + (ga * share).sum(1, keepdim=True)) / total
        if score == "sigmoid":
            q = w * torch.sigmoid(-l).gather(1, idx)
            d, mag = zeros.scatter(1, idx, g * q), zeros.scatter(1, idx, ga * q)
        elif renorm:
            d, mag = zeros.scatter(1, idx, g * w), zeros.scatter(1, idx, ga * w)
        else:
            d = zeros.scatter(1, idx, g * w) - p * (g * w).sum(1, keepdim=True)
            mag = zeros.scatter(1, idx, ga * w) + p * (ga * w).sum(1, keepdim=True)
        out["dlogits"], out["mag"] = torch.where(live, d, 0.0), mag
    return out


def _run(ops, logits, topk, score="softmax", bias=None, groups=1, group_topk=1, renorm=True, scale=1.0, mask=None, dprobs=None):
    x = logits.detach().requires_grad_(dprobs is not None)
    probs, idx, counts = ops.topk_routing(x, topk, score_function=score, expert_bias=bias, num_groups=groups if groups > 1 else None,
                                          group_topk=group_topk if groups > 1 else None, renormalize=renorm, scaling_factor=scale, token_mask=mask)
    out = {"probs": probs.detach(), "indices": idx, "counts": counts}
    if dprobs is not None:
        (out["dlogits"],) = torch.autograd.grad(probs, x, dprobs)
    return out


def _check(got, want, dtype=torch.float32):
    assert got["probs"].dtype == torch.float32 and got["indices"].dtype == torch.int64 and got["counts"].dtype == torch.int64
    assert torch.equal(got["indices"].cpu(), want["indices"])
    assert torch.equal(got["counts"].cpu(), want["counts"])
    err = (got["probs"].double().cpu() - want["probs"]).abs()
    assert bool((err <= 2.0 ** -17 * want["probs"].abs() + 1e-37).all()), float((err / (want["probs"].abs() + 1e-37)).max())
    if "dlogits" in want:
        assert got["dlogits"].dtype == dtype
        fin = torch.finfo(dtype)
        err = (got["dlogits"].double().cpu() - want["dlogits"]).abs()
        bound = 2.0 ** -15 * want["mag"] + fin.eps / 2 * want["dlogits"].abs() + fin.smallest_normal * fin.eps
        assert bool((err <= bound).all()), float((err / bound).max())


def _inputs(gpu, t, e, k, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(t, e, generator=gen) * 1.5).to(dtype).to(gpu)
    bias = (torch.randn(e, generator=gen) * 0.05).to(gpu)
    dprobs = torch.randn(t, k, generator=gen).to(gpu)
    mask = (torch.rand(t, generator=gen) < 0.8).to(gpu)
    return logits, bias, dprobs, mask


SIZES = [(8200, 8, 2), (8193, 63, 7), (1, 1, 1), (1, 2, 1), (3, 7, 7), (65, 8, 2), (130, 16, 3), (33, 20, 12), (70, 32, 4), (9, 33, 32), (50, 64, 6), (21, 64, 17),
         (40, 100, 5), (77, 128, 4), (200, 160, 6), (37, 256, 8), (1, 257, 2), (20, 512, 10), (11, 1000, 32), (5, 1024, 1)]


@pytest.mark.parametrize("t,e,k", SIZES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_choice_probabilities_and_gradient(gpu, t, e, k, score, renorm):
    from primus_amd.pytorch import ops

    for n, (name, dtype) in enumerate(DTYPES.items()):
        for with_bias in (False, True):
            logits, bias, dprobs, mask = _inputs(gpu, t, e, k, dtype, 100 * t + e + n)
            how = dict(score=score, bias=bias if with_bias else None, renorm=renorm, scale=2.5 if with_bias else 1.0, mask=mask if with_bias else None, dprobs=dprobs)
            _check(_run(ops, logits, k, **how), _reference(logits, k, **how), dtype)


GROUPED = [(64, 256, 8, 8, 4), (31, 256, 8, 8, 2), (20, 160, 6, 8, 3), (17, 24, 3, 3, 2), (9, 1023, 8, 33, 4), (13, 60, 5, 5, 5), (7, 64, 2, 64, 7),
           (25, 128, 16, 2, 1), (10, 99, 9, 9, 9), (6, 8, 4, 4, 2), (12, 1024, 32, 16, 4)]


@pytest.mark.parametrize("t,e,k,groups,group_topk", GROUPED)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_groups(gpu, t, e, k, groups, group_topk, score, with_bias):
    from primus_amd.pytorch import ops

    for dtype in (torch.float32, torch.bfloat16):
        logits, bias, dprobs, mask = _inputs(gpu, t, e, k, dtype, t + e + k)
        how = dict(score=score, bias=bias if with_bias else None, groups=groups, group_topk=group_topk, renorm=not with_bias, scale=1.5, dprobs=dprobs, mask=mask)
        _check(_run(ops, logits, k, **how), _reference(logits, k, **how), dtype)


@pytest.mark.parametrize("e,k", [(8, 2), (64, 8), (256, 8), (1024, 32)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_ties_go_to_the_lower_index(gpu, e, k, with_bias):
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(e)
    logits = torch.randint(0, 3, (300, e), generator=gen).float()
    logits[::7] = 0.0
    logits[1::7] = -0.0
    bias = torch.randint(0, 2, (e,), generator=gen).float() * 0.25
    how = dict(score="sigmoid", bias=bias.to(gpu) if with_bias else None)
    _check(_run(ops, logits.to(gpu), k, **how), _reference(logits, k, **how))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,group_topk", [(1, 1), (8, 4)])
@pytest.mark.parametrize("e", [32, 256])
def test_scores_nearer_than_fp32_can_tell(gpu, score, groups, group_topk, e):
    """The bias takes every score to about the same value: the choice hangs on what rounding an fp32 sum loses."""
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(e + groups)
    row = torch.randn(e, generator=gen)
    p = torch.sigmoid(row.double()) if score == "sigmoid" else torch.softmax(row.double(), 0)
    bias = (0.5 - p).float()
    logits = (row + torch.randint(-2, 3, (200, e), generator=gen) * 2.0 ** -23)
    order = (torch.sigmoid(logits.double()) if score == "sigmoid" else torch.softmax(logits.double(), 1)) + bias.double()
    in_fp32 = ((torch.sigmoid(logits) if score == "sigmoid" else torch.softmax(logits, 1)) + bias).topk(4, dim=1).indices
    assert not torch.equal(in_fp32, order.topk(4, dim=1).indices)       # fp32 does lose it
    how = dict(score=score, bias=bias.to(gpu), groups=groups, group_topk=group_topk)
    _check(_run(ops, logits.to(gpu), 4, **how), _reference(logits, 4, **how))


def test_logits_of_disabled_experts_and_of_the_lowest_value(gpu):
    """-inf, the type's lowest value and rows that have nothing else; what is not finite stays in its row."""
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(4)
    for dtype in DTYPES.values():
        logits = torch.randn(40, 96, generator=gen).to(dtype)
        logits[:, ::3] = -math.inf
        logits[5:20, 1::3] = torch.finfo(dtype).min
        logits[20:25, 8:] = -math.inf                                # fewer finite ones than are chosen
        for score in ("softmax", "sigmoid"):
            for bias in (None, torch.randn(96, generator=gen)):
                how = dict(score=score, bias=None if bias is None else bias.to(gpu))
                _check(_run(ops, logits.to(gpu), 6, **how), _reference(logits, 6, **how))


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("groups", [1, 4])
def test_rows_of_disabled_experts_alone_give_zeros(gpu, renorm, groups):
    from primus_amd.pytorch import ops

    x = torch.full((70, 32), -math.inf, device=gpu)
    x[1::2] = torch.arange(32.0, device=gpu)
    x.requires_grad_()
    for bias in (None, torch.randn(32, device=gpu)):
        for score in ("softmax", "sigmoid"):
            probs, idx, _ = ops.topk_routing(x, 4, score_function=score, expert_bias=bias, renormalize=renorm, num_groups=groups if groups > 1 else None,
                                             group_topk=2 if groups > 1 else None)
            (dx,) = torch.autograd.grad(probs, x, torch.ones_like(probs))
            assert not bool(probs[::2].any()) and not bool(dx[::2].any()) and bool(torch.isfinite(probs).all()) and bool(torch.isfinite(dx).all())
            assert all(len(set(r)) == 4 and min(r) >= 0 and max(r) < 32 for r in idx.tolist())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_rows_that_are_not_finite_keep_valid_indices(gpu, score, bias, groups):
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(6)
    logits = torch.randn(64, 64, generator=gen)
    clean = logits.clone()
    logits[3] = math.nan
    logits[7, 5] = math.nan
    logits[11, 9] = math.inf
    logits[13] = -math.inf
    logits[17] = math.inf
    b = torch.randn(64, generator=gen).to(gpu) * 0.1 if bias else None
    probs, idx, counts = ops.topk_routing(logits.to(gpu), 6, score_function=score, expert_bias=b, num_groups=groups if groups > 1 else None,
                                          group_topk=2 if groups > 1 else None)
    assert bool(((idx >= 0) & (idx < 64)).all()) and int(counts.sum()) == idx.numel()
    assert all(len(set(r)) == 6 for r in idx.tolist())
    ok = [i for i in range(64) if i not in (3, 7, 11, 13, 17)]
    want = _reference(clean, 6, score=score, bias=b, groups=groups, group_topk=2 if groups > 1 else 1)
    assert torch.equal(idx.cpu()[ok], want["indices"][ok])
    # a masked row may hold anything
    mask = torch.ones(64, dtype=torch.bool)
    mask[[3, 7, 11, 13, 17]] = False
    x = logits.to(gpu).requires_grad_()
    probs, idx, counts = ops.topk_routing(x, 6, score_function=score, expert_bias=b, token_mask=mask.to(gpu))
    (dx,) = torch.autograd.grad(probs, x, torch.ones_like(probs))
    assert bool(torch.isfinite(probs).all()) and bool(torch.isfinite(dx).all()) and not bool(dx[~mask.to(gpu)].any())
    assert bool((idx[~mask.to(gpu)] == -1).all()) and int(counts.sum()) == 59 * 6


@pytest.mark.parametrize("t", [0, 1, 128, 256, 257, 4097, 50000])
def test_counts_over_one_and_many_workgroups(gpu, t):
    from primus_amd.pytorch import ops

    gen = torch.Generator(device=gpu).manual_seed(t)
    logits = torch.randn(t, 24, generator=gen, device=gpu)
    mask = torch.rand(t, generator=gen, device=gpu) < 0.7
    probs, idx, counts = ops.topk_routing(logits, 3, token_mask=mask)
    want = torch.topk(logits, 3, dim=1).indices       # no ties among 24 random floats a row, checked here
    assert bool((logits.sort(dim=1).values.diff(dim=1) > 0).all())
    assert torch.equal(idx, torch.where(mask[:, None], want, -1))
    assert torch.equal(counts, torch.bincount(want[mask].reshape(-1), minlength=24))
    assert probs.shape == (t, 3)


def test_gradient_against_differences(gpu):
    """Central differences of the fp64 definition are not the kernel's, so the kernel's own probabilities are differenced: a step of
    2^-9 leaves an error of about h^2 f''' / 6 < 2^-18 and of 2^-23 / h = 2^-14 from the rounding of the two values."""
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(12)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            logits = torch.randn(6, 12, generator=gen).to(gpu)
            g = torch.randn(6, 3, generator=gen).to(gpu)
            x = logits.clone().requires_grad_()
            probs, idx, _ = ops.topk_routing(x, 3, score_function=score, renormalize=renorm)
            (dx,) = torch.autograd.grad(probs, x, g)
            h = 2.0 ** -9
            for e in range(12):
                up, down = logits.clone(), logits.clone()
                up[:, e] += h
                down[:, e] -= h
                pu, iu, _ = ops.topk_routing(up, 3, score_function=score, renormalize=renorm)
                pd, idn, _ = ops.topk_routing(down, 3, score_function=score, renormalize=renorm)
                same = (iu == idx).all(1) & (idn == idx).all(1)
                diff = ((pu.double() - pd.double()) * g.double()).sum(1) / (2 * h)
                assert bool(((dx[:, e].double() - diff).abs()[same] <= 2.0 ** -12).all())


def test_strides_and_other_streams(gpu):
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(64, 80, generator=gen).to(gpu)
    logits = wide[:, 5:69].t().contiguous().t()        # column-major view
    want = _reference(logits, 4)
    _check(_run(ops, logits, 4), want)
    _check(_run(ops, wide[:, 5:69], 4), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(ops, logits, 4)
    torch.cuda.current_stream().wait_stream(side)
    _check(got, want)
