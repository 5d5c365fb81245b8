"""Gradient norm and clipping under Megatron's names: what they hand to the operators, ranks' norms put together over gloo, and the patch."""

import math
import os
from types import SimpleNamespace

import pytest
import torch

from primus_amd.megatron.optimizer import clip_grads
from primus_amd.megatron.patches import apply_patches, registered_patches
from primus_amd.pytorch import ops


def _norm(grads, kind=2.0):
    """The operator's definition on the CPU."""
    flat = torch.cat([g.double().reshape(-1) for g in grads])
    return (flat.abs().max() if kind == math.inf else flat.norm()).float()


def _rank(rank, world, port, kind, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    torch.distributed.init_process_group("gloo", rank=rank, world_size=world)
    ops.grad_norm = _norm
    grads = [torch.full((3,), 3e25 * (rank + 1)), torch.tensor([-4e25])]
    total = clip_grads.get_grad_norm_fp32(grads, kind, torch.distributed.group.WORLD)
    alone = clip_grads.get_grad_norm_fp32(grads, kind)
    out.put((rank, total.item(), alone.item(), total.dtype == torch.float32 and total.dim() == 0))
    torch.distributed.destroy_process_group()


@pytest.mark.parametrize("kind", [2, math.inf])
def test_norm_over_two_ranks(kind):
    """The norm of both ranks' gradients; their squares would not fit a float32."""
    ctx = torch.multiprocessing.get_context("spawn")
    out = ctx.SimpleQueue()
    port = 29600 + os.getpid() % 300 + (7 if kind == 2 else 0)
    ranks = [ctx.Process(target=_rank, args=(r, 2, port, kind, out)) for r in range(2)]
    for r in ranks:
        r.start()
    got = sorted(out.get() for _ in ranks)
    for r in ranks:
        r.join()
        assert r.exitcode == 0
    every = [[3e25 * (r + 1)] * 3 + [-4e25] for r in range(2)]
    norm = (lambda v: max(map(abs, v))) if kind == math.inf else (lambda v: math.sqrt(math.fsum(x * x for x in v)))
    for rank, total, alone, scalar in got:
        # (each rank's norm is rounded to fp32, and so is the total: half a step each, and the inputs' own)
        assert scalar and abs(total - norm(every[0] + every[1])) <= 3 * 2.0 ** -24 * total
        assert abs(alone - norm(every[rank])) <= 2 * 2.0 ** -24 * alone


def test_which_gradients_are_clipped(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, "clip_grads", lambda grads, max_norm, norm: seen.append((grads, max_norm, norm)))
    ps = [torch.nn.Parameter(torch.zeros(n)) for n in (2, 3, 4)]
    ps[0].grad, ps[2].grad = torch.ones(2), torch.ones(4)
    ps[1].decoupled_grad = torch.ones(3)
    norm = torch.tensor(2.0)
    clip_grads.clip_grad_by_total_norm_fp32(ps, 1.0, norm)
    clip_grads.clip_grad_by_total_norm_fp32(iter(ps), 1.0, 2.5, use_decoupled_grad=True)
    clip_grads.clip_grad_by_total_norm_fp32(ps[0], 3, norm)
    clip_grads.clip_grad_by_total_norm_fp32(ps[1], 3, norm)        # no gradient: nothing to do
    assert len(seen) == 3
    assert [g.data_ptr() for g in seen[0][0]] == [ps[0].grad.data_ptr(), ps[2].grad.data_ptr()] and seen[0][1:] == (1.0, norm)
    assert [g.data_ptr() for g in seen[1][0]] == [ps[1].decoupled_grad.data_ptr()] and seen[1][1:] == (1.0, 2.5)
    assert [g.data_ptr() for g in seen[2][0]] == [ps[0].grad.data_ptr()]


def test_patch():
    assert "megatron.optimizer.clip_grads" in registered_patches()
    paths = ["megatron.core.optimizer.clip_grads", "megatron.core.optimizer.optimizer", "megatron.core.extensions.transformer_engine_spec_provider",
             "megatron.core.models.gpt.gpt_layer_specs", "megatron.core.models.gpt.moe_module_specs", "megatron.core.transformer.multi_token_prediction"]
    for on, turbo in ((True, True), (False, True), (True, False)):
        targets = {p: SimpleNamespace() for p in paths}
        apply_patches(SimpleNamespace(enable_primus_turbo=turbo, use_turbo_clip_grads=on), targets)
        for path in paths[:2]:
            assert (getattr(targets[path], "get_grad_norm_fp32", None) is clip_grads.get_grad_norm_fp32) == (on and turbo)
            assert (getattr(targets[path], "clip_grad_by_total_norm_fp32", None) is clip_grads.clip_grad_by_total_norm_fp32) == (on and turbo)
