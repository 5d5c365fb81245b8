"""The norm over ranks: a NaN of one rank, whatever its place, and which ranks a group of None means.  Two processes over gloo."""

import math
import os

import pytest
import torch

from primus_amd.megatron.optimizer import clip_grads
from primus_amd.pytorch import ops

CASES = [[1.0, 2.0], [math.nan, 2.0], [2.0, math.nan], [math.nan, math.inf], [math.inf, math.nan], [math.inf, 1.0], [0.0, 0.0], [0.0, 1e-45], [3e38, 2e38]]


def _rank(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    torch.distributed.init_process_group("gloo", rank=rank, world_size=world)
    ops.grad_norm = lambda grads, kind=2.0: grads[0].abs().max()
    group = torch.distributed.group.WORLD
    for values in CASES:
        grads = [torch.tensor([values[rank]])]
        top = clip_grads.get_grad_norm_fp32(grads, math.inf, group)
        out.put((rank, top.item(), clip_grads.get_grad_norm_fp32(grads, 2, group).item(), clip_grads.get_grad_norm_fp32(grads, math.inf, grad_stats_parallel_group=None).item(),
                 clip_grads.get_grad_norm_fp32(grads, grad_stats_parallel_group=None).item(), clip_grads.get_grad_norm_fp32(grads).item(),
                 top.dtype == torch.float32 and top.dim() == 0))
    torch.distributed.destroy_process_group()


@pytest.fixture(scope="module")
def norms():
    """``{rank: [(largest, 2-norm, and both for a group of None, of the rank alone), ...]}``"""
    ctx = torch.multiprocessing.get_context("spawn")
    out = ctx.SimpleQueue()
    port = 29950 + os.getpid() % 300
    ranks = [ctx.Process(target=_rank, args=(r, 2, port, out)) for r in range(2)]
    for r in ranks:
        r.start()
    got = {0: [], 1: []}
    for _ in range(2 * len(CASES)):
        rank, *values = out.get()
        got[rank].append(values)
    for r in ranks:
        r.join()
        assert r.exitcode == 0
    return got


def _same(a, b):
    return math.isnan(a) and math.isnan(b) or a == b or abs(a - b) <= 2 * 2.0 ** -24 * abs(b)


@pytest.mark.parametrize("at", range(len(CASES)))
def test_largest_magnitude(norms, at):
    """NaN where any rank has one."""
    want = math.nan if any(map(math.isnan, CASES[at])) else torch.tensor(max(CASES[at])).item()
    for rank in (0, 1):
        top, *_, scalar = norms[rank][at]
        assert scalar and (top == want or math.isnan(top) and math.isnan(want)), (rank, top)


def _of_all(values):
    return math.nan if any(map(math.isnan, values)) else torch.tensor(math.hypot(*torch.tensor(values).tolist())).item()


@pytest.mark.parametrize("at", range(len(CASES)))
def test_which_ranks(norms, at):
    """A group, None for all ranks, and the rank alone where none is named."""
    for rank in (0, 1):
        top, two, every_top, every_two, alone, _ = norms[rank][at]
        assert _same(two, _of_all(CASES[at])) and _same(every_two, two) and _same(every_top, top)
        assert _same(alone, torch.tensor(CASES[at][rank]).item())


def test_without_ranks(monkeypatch):
    assert not torch.distributed.is_initialized()
    monkeypatch.setattr(ops, "grad_norm", lambda grads, kind=2.0: grads[0].abs().max())
    for kind in (2, math.inf):
        assert clip_grads.get_grad_norm_fp32([torch.tensor([-3.0])], kind, None).item() == 3.0
