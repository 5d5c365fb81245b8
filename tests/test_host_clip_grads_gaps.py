"""Clipping's refusals of tensors with gaps that overlap what is written, and that slices beside each other are let through: checked without a GPU."""

import itertools

import pytest
import torch

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


def _b(*shape):
    return torch.zeros(*(shape or (10, 12)))


def _calls():
    b, s, w, c = _b(), torch.zeros(6, 6), torch.zeros(4, 6, 8), torch.zeros(200)
    ones = lambda *a: [torch.ones_like(t, memory_format=torch.contiguous_format) for t in a]  # noqa: E731
    yield "columns", [b[:, 0:5], b[:, 3:8]], None, None
    yield "rows and columns", [b[2:6, 0:5], b[4:9, 4:8]], None, None
    yield "every other row", [b[::2, :7], b[::4]], None, None
    yield "a tensor and its transpose", ones(s, s), [s, s.t()], None
    yield "a slice of an output", ones(s, s[:, 1:3]), [s, s[:, 1:3]], None
    yield "a gradient that is read", [b[:, 2:6]], [b[:, 4:8]], None
    yield "a dense gradient that is read", [c[:24].view(4, 6)], [c[20:68].view(4, 12)[:, :6]], None
    yield "a gradient with gaps and a dense output", [s.t()], [s], None
    yield "the norm in a column", [b[:, :3]], None, b[0, 1]
    yield "the norm in the last element", [b[:, 3:]], None, b[9, 11]
    yield "the norm in an output", ones(b[:, :3]), [b[:, :3]], b[4, 2:3]
    yield "itself, by strides", [c.as_strided((4, 4), (2, 3))], None, None
    yield "itself, windows", [c.unfold(0, 8, 4)], None, None
    yield "itself, expanded", [_b(1, 3).expand(2, 3)], None, None
    yield "three dimensions", [w[:, 0:3, 0:5], w[:, 2:4, 4:8]], None, None
    yield "types", [b[:, 0:4]], [b.view(torch.bfloat16)[:, 6:10]], None


@pytest.mark.parametrize("what,grads,out,norm", list(_calls()), ids=lambda v: v if isinstance(v, str) else "")
def test_overlaps_are_refused(what, grads, out, norm):
    with pytest.raises(ValueError, match="overlap"):
        ops.clip_grads(grads, 1.0, norm=norm, out=out)


def _apart():
    b, s, w, c = _b(), torch.zeros(6, 6), torch.zeros(4, 6, 8), torch.zeros(200)
    ones = lambda *a: [torch.ones_like(t, memory_format=torch.contiguous_format) for t in a]  # noqa: E731
    yield "columns", [b[:, 0:5], b[:, 5:8], b[:, 8:]], None, None
    yield "columns of a transpose", [b.t()[0:5], b.t()[5:8]], None, None
    yield "blocks", [b[:5, :6], b[:5, 6:], b[5:, :6], b[5:, 6:]], None, None
    yield "rows in turn", [b[::2, 1:], b[1::2, 1:]], None, None
    yield "columns in turn", [b[:, ::2], b[:, 1::2]], None, None
    yield "the norm between", [b[:, :3]], None, b[0, 3]
    yield "the norm behind", [b[:, 3:11]], None, b[9, 11]
    yield "three dimensions", [w[:, 0:2, 0:4], w[:, 0:2, 4:8], w[:, 2:, :4], w[:, 2:, 4:]], None, None
    yield "steps across", [w[:, 0:2, 2:4], w[:, 1:3, 0:2]], None, None
    yield "halves", [w.view(4, 2, 3, 8)[:, 0], w.view(4, 2, 3, 8)[:, 1]], None, None
    yield "its own output", [b[:, 3:7]], [b[:, 3:7]], None
    yield "a gradient twice", [b[:, 3:7], b[:, 3:7]], ones(b[:, 3:7], b[:, 3:7]), None
    yield "no elements", [b[:, 3:3], b[:, 1:5]], None, None
    yield "a column of one", [b[:, 0:1], b[:, 1:2]], None, None


@pytest.mark.parametrize("what,grads,out,norm", list(_apart()), ids=lambda v: v if isinstance(v, str) else "")
def test_slices_beside_each_other_are_not(what, grads, out, norm):
    with pytest.raises(Launched):
        ops.clip_grads(grads, 1.0, norm=norm, out=out)


def test_spans_against_the_elements():
    """All pairs of slices of a small tensor: those that share an element meet by the rule."""
    base = torch.arange(4 * 6, dtype=torch.int32).view(4, 6)
    cuts = [slice(a, b, st) for st in (1, 2) for a, b in ((0, 4), (0, 2), (1, 3), (2, 6), (3, 4))]
    views = [base[r, c] for r, c in itertools.product(cuts, cuts)]
    views = [v for v in views + [v.t() for v in views[::7]] if v.numel()]
    for a, b in itertools.combinations(views, 2):
        shared = set(a.flatten().tolist()) & set(b.flatten().tolist())
        assert not shared or not ops._apart([ops._span(a, True), ops._span(b, True)]), (a, b)
