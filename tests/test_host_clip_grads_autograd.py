"""The gradient norm and clipping are outside autograd: tangents and traces are refused instead of being dropped, and plain tensors beside a tangent are not."""

import pytest
import torch
from torch.autograd import forward_ad

from primus_amd.pytorch import kernels as K
from primus_amd.pytorch import ops


class Launched(Exception):
    pass


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    def launch(*a, **k):
        raise Launched

    monkeypatch.setattr(K, "grad_norm_impl", launch)
    monkeypatch.setattr(K, "clip_grads_impl", launch)


def _calls(t, plain):
    return {"norm": lambda: ops.grad_norm(t), "norm of a list": lambda: ops.grad_norm([plain, t]), "norm of a slice": lambda: ops.grad_norm([t[:, :2]]),
            "clip": lambda: ops.clip_grads([plain, t], 1.0), "clip from": lambda: ops.clip_grads([t], 1.0, out=[plain]),
            "clip into": lambda: ops.clip_grads([plain], 1.0, out=[t]), "clip a slice": lambda: ops.clip_grads([t[:, :2]], 1.0),
            "clip by": lambda: ops.clip_grads([plain], 1.0, norm=t.sum())}


@pytest.mark.parametrize("name", list(_calls(None, None)))
def test_tangents_are_refused(name):
    with forward_ad.dual_level():
        t = forward_ad.make_dual(torch.ones(3, 4), torch.ones(3, 4))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _calls(t, torch.ones(3, 4))[name]()
        with pytest.raises(Launched):
            _calls(torch.ones(3, 4), torch.ones(3, 4))[name]()


@pytest.mark.filterwarnings("ignore::DeprecationWarning", "ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", list(_calls(None, None)))
def test_traces_are_refused(name):
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(lambda t: _calls(t, torch.ones(3, 4))[name](), (torch.ones(3, 4),), check_trace=False)


def test_gradients_with_a_graph_are_taken_as_they_are():
    """As under ``torch.no_grad``."""
    w = torch.ones(3, 4, requires_grad=True)
    for t in (w, w * 2):
        for call in _calls(t, torch.ones(3, 4)).values():
            with pytest.raises(Launched):
                call()
