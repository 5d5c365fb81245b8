"""Gradient norm and clipping under the names that Megatron-LM's optimizers import (``megatron.core.optimizer.clip_grads``), on the
operators of this package: every gradient is read once for the norm and the factor stays on the device, so a step does not
wait for the host.  Gradients are plain tensors; of sharded ones (DTensor) the caller hands in the local parts.  ``patches/turbo.py``
installs both with ``use_turbo_clip_grads``.
"""

from __future__ import annotations

import math
from typing import Iterable, List, Optional, Union

import torch

from ...pytorch import ops


_THIS_RANK = object()


@torch.no_grad()
def get_grad_norm_fp32(grads_for_norm: Union[List[torch.Tensor], torch.Tensor], norm_type: Union[int, float] = 2,
                       grad_stats_parallel_group: Optional["torch.distributed.ProcessGroup"] = _THIS_RANK) -> torch.Tensor:
    """Norm of the gradients of all ranks of ``grad_stats_parallel_group``, 2 or inf.  None is the default group, every rank, as ``torch.distributed`` and
    Megatron-LM have it, whose distributed optimizer hands None over for that (with one process and no group, this rank's norm); left out, this
    rank's alone.  A float32 scalar on the device, which formats and compares like the number it stands for.  Between the ranks squares are added in
    float64; the largest magnitude is NaN if any rank's is."""
    norm = ops.grad_norm(grads_for_norm, float(norm_type))
    if grad_stats_parallel_group is _THIS_RANK or (grad_stats_parallel_group is None and not torch.distributed.is_initialized()):
        return norm
    if float(norm_type) == math.inf:
        # (of numbers that are not negative the bits are ordered as they are, and a NaN's are above all; a maximum of floats may lose it)
        torch.distributed.all_reduce(norm.view(torch.int32), op=torch.distributed.ReduceOp.MAX, group=grad_stats_parallel_group)
        return norm
    total = norm.double().square()
    torch.distributed.all_reduce(total, op=torch.distributed.ReduceOp.SUM, group=grad_stats_parallel_group)
    return total.sqrt().float()


def clip_grad_by_total_norm_fp32(parameters: Union[Iterable[torch.Tensor], torch.Tensor], max_norm: Union[int, float],
                                 total_norm: Union[torch.Tensor, float], use_decoupled_grad: bool = False) -> None:
    """Scales the parameters' gradients (``decoupled_grad`` or ``grad``; parameters without one are left out) in place by
    ``min(1, max_norm / (total_norm + 1e-6))``."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [getattr(p, "decoupled_grad", None) if use_decoupled_grad else p.grad for p in parameters]
    grads = [g.detach() for g in grads if g is not None]
    if grads:
        ops.clip_grads(grads, max_norm, norm=total_norm)
