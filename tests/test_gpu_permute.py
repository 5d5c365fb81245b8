"""``ops.permute_tokens`` / ``ops.unpermute_tokens`` against index arithmetic on the host: rows, probabilities, lengths and the
permutation are equal bit for bit; sums are compared with 64-bit ones.

Tolerance of a sum of K products in fp32, rounded once: (K + 1) 2^-24 of the sum of magnitudes plus half a step of the type.  A
dot product over H elements in fp32 (at most H / 64 + 8 additions in a row, products fused): (H / 64 + 10) 2^-24 of the sum of magnitudes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _plan(indices, experts, align):
    """Entry after entry, as the definition says."""
    flat = indices.reshape(-1).tolist()
    rows = (len(flat) + experts * (align - 1)) // align * align
    at, lens, row_of, entry_of = 0, [], [-1] * len(flat), [-1] * rows
    by = [[] for _ in range(experts)]
    for i, e in enumerate(flat):
        if 0 <= e < experts:
            by[e].append(i)
    for mine in by:
        for j, i in enumerate(mine):
            row_of[i], entry_of[at + j] = at + j, i
        n = -(-len(mine) // align) * align
        lens.append(n)
        at += n
    lens[-1] += rows - at
    return torch.tensor(row_of).view(indices.shape), torch.tensor(entry_of, dtype=torch.int32), torch.tensor(lens)


def _indices(t, k, experts, gen, dropped=0.1):
    idx = torch.randint(0, experts, (t, k), generator=gen)
    idx[torch.rand(t, k, generator=gen) < dropped] = -1
    return idx


def _check(ops, gpu, idx, experts, align, hidden, dtype, probs_dtype, gen, with_grad=True):
    t, k = idx.shape
    row_of, entry_of, lens = _plan(idx, experts, align)
    rows = entry_of.numel()
    live, token = entry_of >= 0, (entry_of // k).clamp(min=0).long()
    x = torch.randn(t, hidden, generator=gen).to(dtype)
    probs = None if probs_dtype is None else torch.rand(t, k, generator=gen).to(probs_dtype)
    xd = x.to(gpu).requires_grad_()
    pd = None if probs is None else probs.to(gpu).requires_grad_()
    got, got_probs, got_lens, perm = ops.permute_tokens(xd, idx.to(gpu), experts, probs=pd, align=align)
    assert torch.equal(perm.row_of.cpu(), row_of) and torch.equal(perm.entry_of.cpu(), entry_of) and torch.equal(got_lens.cpu(), lens)
    assert got.shape == (rows, hidden) and got.dtype == dtype
    want = torch.where(live[:, None], x[token], 0.0) if t else x.new_zeros(rows, hidden)
    assert torch.equal(got.detach().cpu(), want)
    if probs is not None:
        assert torch.equal(got_probs.detach().cpu(), torch.where(live, probs.reshape(-1)[entry_of.clamp(min=0).long()], 0.0) if t else probs.new_zeros(rows))
    if not with_grad or not t:
        return
    half = torch.finfo(dtype).eps / 2
    drows = torch.randn(rows, hidden, generator=gen).to(dtype)
    on = (row_of >= 0)
    part = torch.where(on[:, :, None], drows[row_of.clamp(min=0)].double(), 0.0)
    if probs is None:
        grads = torch.autograd.grad(got, xd, drows.to(gpu))
    else:
        dprobs_in = torch.randn(rows, generator=gen).to(probs_dtype)
        grads = torch.autograd.grad([got, got_probs], [xd, pd], [drows.to(gpu), dprobs_in.to(gpu)])
        assert torch.equal(grads[1].cpu(), torch.where(on, dprobs_in[row_of.clamp(min=0)], 0.0))
    dx = part.sum(1)
    assert bool(((grads[0].double().cpu() - dx).abs() <= (k + 1) * 2.0 ** -24 * part.abs().sum(1) + half * dx.abs() + 1e-30).all())

    # back: rows that no entry went to hold what must not be seen
    y_rows = torch.randn(rows, hidden, generator=gen).to(dtype)
    y_rows[~live] = float("nan")
    rd = y_rows.to(gpu).requires_grad_()
    w = torch.ones(t, k, dtype=torch.float64) if probs is None else probs.double()
    part = torch.where(on[:, :, None], y_rows[row_of.clamp(min=0)].double(), 0.0)
    y = ops.unpermute_tokens(rd, perm, probs=pd)
    want = (part * w[:, :, None]).sum(1)
    assert bool(((y.detach().double().cpu() - want).abs() <= (k + 1) * 2.0 ** -24 * (part.abs() * w[:, :, None]).sum(1) + half * want.abs() + 1e-30).all())
    dy = torch.randn(t, hidden, generator=gen).to(dtype)
    grads = torch.autograd.grad(y, [rd] if probs is None else [rd, pd], dy.to(gpu))
    want = torch.where(live[:, None], dy[token].double() * w.reshape(-1)[entry_of.clamp(min=0).long()][:, None], 0.0)
    assert bool(((grads[0].double().cpu() - want).abs() <= (half + 2.0 ** -24) * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all())
    if probs is not None:
        terms = part * dy.double()[:, None, :]
        want = terms.sum(2)
        bound = (hidden / 64 + 10) * 2.0 ** -24 * terms.abs().sum(2) + torch.finfo(probs_dtype).eps / 2 * want.abs() + 1e-30
        assert grads[1].dtype == probs_dtype and bool(((grads[1].double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("t,k,experts", [(0, 2, 3), (1, 1, 1), (1, 8, 128), (7, 3, 5), (64, 2, 8), (129, 4, 1024), (333, 6, 32), (700, 8, 100)])
@pytest.mark.parametrize("align", [1, 16, 32])
def test_small(gpu, t, k, experts, align):
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(1000 * t + experts + align)
    for n, (hidden, dtype) in enumerate([(64, torch.bfloat16), (1, torch.float32), (33, torch.float16), (520, torch.bfloat16), (77, torch.bfloat16), (1028, torch.float32)]):
        _check(ops, gpu, _indices(t, k, experts, gen), experts, align, hidden, dtype, (None, torch.float32, torch.bfloat16, torch.float16)[n % 4], gen)


@pytest.mark.parametrize("t,k,experts,align", [(5000, 2, 8, 1), (3001, 8, 256, 32), (40000, 4, 3, 1), (140000, 8, 61, 16)])
def test_many_workgroups(gpu, t, k, experts, align):
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(t)
    _check(ops, gpu, _indices(t, k, experts, gen), experts, align, 24, torch.bfloat16, torch.float32, gen)


@pytest.mark.parametrize("case", ["one_expert", "nothing_routed", "same_expert_twice", "out_of_range", "ascending", "descending"])
def test_edge_routings(gpu, case):
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(8)
    t, k, experts = 300, 4, 17
    idx = {"one_expert": torch.full((t, k), 16), "nothing_routed": torch.full((t, k), -1), "same_expert_twice": torch.tensor([[3, 3, 5, 3]]).repeat(t, 1),
           "out_of_range": torch.randint(-40, 60, (t, k), generator=gen), "ascending": (torch.arange(t * k) * experts // (t * k)).view(t, k),
           "descending": (experts - 1 - torch.arange(t * k) * experts // (t * k)).view(t, k)}[case]
    if case == "out_of_range":
        idx[5, 2], idx[6, 1] = 1 << 40, -(1 << 62)
    for align in (1, 32):
        _check(ops, gpu, idx, experts, align, 40, torch.bfloat16, torch.float32, gen)


def test_rows_off_their_alignment_and_strided(gpu):
    """Storage that starts between two 16-byte boundaries, and views whose rows are apart."""
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(2)
    idx = _indices(50, 3, 6, gen).to(gpu)
    flat = torch.randn(50 * 64 + 8, generator=gen).bfloat16().to(gpu)
    for x in (flat[1:1 + 50 * 64].view(50, 64), flat[4:4 + 50 * 64].view(50, 64), torch.randn(50, 100, generator=gen).bfloat16().to(gpu)[:, 9:73]):
        a = ops.permute_tokens(x, idx, 6)
        b = ops.permute_tokens(x.clone(memory_format=torch.contiguous_format), idx, 6)
        assert torch.equal(a[0], b[0])
        rows = torch.empty(a[0].numel() + 8, dtype=torch.bfloat16, device=gpu)[1:1 + a[0].numel()].view_as(a[0]).copy_(a[0])
        assert torch.equal(ops.unpermute_tokens(rows, a[3]), ops.unpermute_tokens(a[0], a[3]))


def test_only_some_gradients_are_asked_for(gpu):
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(5)
    idx = _indices(40, 2, 6, gen).to(gpu)
    x, p = torch.randn(40, 32, generator=gen).to(gpu), torch.rand(40, 2, generator=gen).to(gpu)
    rows, row_probs, _, perm = ops.permute_tokens(x, idx, 6, probs=p.requires_grad_())
    (only,) = torch.autograd.grad(row_probs.sum(), p)
    assert torch.equal(only, (idx >= 0).float())
    rows = rows.detach()
    dy = torch.randn(40, 32, generator=gen).to(gpu)
    both = torch.autograd.grad(ops.unpermute_tokens(rows.requires_grad_(), perm, probs=p), [rows, p], dy)
    (a,) = torch.autograd.grad(ops.unpermute_tokens(rows, perm, probs=p.detach()), rows, dy)
    (b,) = torch.autograd.grad(ops.unpermute_tokens(rows.detach(), perm, probs=p), p, dy)
    assert torch.equal(a, both[0]) and torch.equal(b, both[1])


def test_more_than_2_to_31_bytes(gpu):
    """Rows past byte offsets of 32 bits."""
    from primus_amd.pytorch import ops

    t, k, hidden, experts = 150000, 2, 8192, 4             # 2.5 GB of tokens, 4.9 GB of rows
    x = (torch.arange(t, device=gpu) % 251).to(torch.bfloat16)[:, None].expand(t, hidden).contiguous()
    idx = torch.stack([torch.arange(t, device=gpu) % experts, (torch.arange(t, device=gpu) + 1) % experts], 1)
    rows, _, lens, perm = ops.permute_tokens(x, idx, experts)
    assert int(lens.sum()) == t * k
    token = (perm.entry_of // k).long()
    assert torch.equal(rows[:, 0], x[token, 0]) and torch.equal(rows[:, -1], x[token, -1])
    assert torch.equal(torch.sort(perm.entry_of).values, torch.arange(t * k, device=gpu, dtype=torch.int32))
    y = ops.unpermute_tokens(rows, perm)
    assert torch.equal(y[:, 0], x[:, 0] * 2) and torch.equal(y[:, -1], x[:, -1] * 2)
