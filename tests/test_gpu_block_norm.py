"""Norms where blocks meet (``ops.add_rmsnorm``, ``ops.rmsnorm_add``) on the GPU against the formulas in float64.

Bars.  u, us: half a step of the type of x and of the residual stream (2^-8 bf16, 2^-11 fp16, 2^-24 fp32), e = 2^-24.  A value is rounded once: u * |v|.
fp32 work before that: a row's sum in lanes and trees of at most 64 additions, and under 16 operations an element, is 64 e of the magnitudes that are
added.  The backward normalises h as it was rounded: us of hh, once in hh itself and once through mean(g hh).  Sums over rows are serial in the worst
case: rows * e more."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
EPS, POST_EPS = 1e-5, 1e-3


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _gate_shape(kind, lead, k):
    return {"": None, "column": (k,), "element": (1,), "scalar": (), "first": (lead[0],) + (1,) * (len(lead) - 1) + (k,), "last": (1,) * (len(lead) - 1) + (lead[-1], k),
            "token": lead + (1,), "full": lead + (k,), "first_scalar": (lead[0],) + (1,) * len(lead)}[kind]


def _inputs(lead, k, dtype, stream, post, gate, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed + 17 * k + sum(lead))
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    v = {"x": n(*lead, k) * torch.logspace(-1, 1, k)[torch.randperm(k, generator=g)], "residual": 2 * n(*lead, k), "weight": 1 + 0.2 * n(k),
         "post_weight": 1 + 0.2 * n(k) if post else None, "gate": None if not gate else 0.5 + 0.5 * n(*_gate_shape(gate, lead, k))}
    v = {name: None if t is None else t.to(stream if name == "residual" else dtype).to(device) for name, t in v.items()}
    return v, n(*lead, k).to(dtype).to(device), n(*lead, k).to(stream).to(device)


def _to(t, shape):
    """Summed over what ``shape`` broadcasts over."""
    dims = [d for d in range(t.dim()) if d < t.dim() - len(shape) or shape[d - t.dim() + len(shape)] == 1 != t.shape[d]]
    return (t.sum(dims) if dims else t).reshape(shape)


def _reference(v, dy, dh, scale, dtype, stream, pre=True, eps=EPS, post_eps=POST_EPS):
    """``{name: (value, bound)}`` in float64 on the CPU."""
    d = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    x, res, w, wp, gate = (d(v[n]) for n in ("x", "residual", "weight", "post_weight", "gate"))
    dy, dh = d(dy), d(dh)
    u, us = _u(dtype), _u(stream)
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    rows = x.numel() // x.shape[-1]
    rp = 1 / torch.sqrt(mean(x * x) + post_eps)
    xh = x * rp
    n = xh * wp if wp is not None else x
    f = scale * gate if gate is not None else torch.tensor(float(scale), dtype=torch.float64)
    h = res + f * n
    mag_h = res.abs() + (f * n).abs()
    out = {"h": (h, us * h.abs() + 64 * E * mag_h)}
    t, big = (torch.zeros_like(h), torch.zeros_like(h)) if dh is None else (dh, dh.abs())
    err = torch.zeros_like(h)
    if pre:
        r = 1 / torch.sqrt(mean(h * h) + eps)
        hh = h * r
        out["y"] = (hh * w, u * (hh * w).abs() + 64 * E * (mag_h * r * w.abs() + (hh * w).abs()))
        if dy is not None:
            g = dy * w
            c1, c1_mag = mean(g * hh), mean((g * hh).abs())
            t = t + r * (g - hh * c1)
            big = big + r * (g.abs() + hh.abs() * c1_mag)
            err = err + 2 * us * r * hh.abs() * c1_mag
            every = (dy * hh).abs().reshape(rows, -1).sum(0)
            dw = (dy * hh).reshape(rows, -1).sum(0)
            out["weight"] = (dw, u * dw.abs() + (us + (64 + rows) * E) * every)
    err = err + 64 * E * big
    out["residual"] = (t, us * t.abs() + err)
    if wp is None:
        dx, dx_err = f * t, f.abs() * err
    else:
        q, a = f * wp * xh, (f * wp * xh).abs()
        c2 = mean(q * t)
        dx = rp * (f * t * wp - xh * c2)
        dx_err = rp * ((f * wp).abs() * err + xh.abs() * mean(a * err)) + 64 * E * rp * ((f * t * wp).abs() + xh.abs() * mean(a * big))
        dwp = (f * t * xh).reshape(rows, -1).sum(0)
        out["post_weight"] = (dwp, u * dwp.abs() + ((f * xh).abs() * (err + (64 + rows) * E * big)).reshape(rows, -1).sum(0))
    out["x"] = (dx, u * dx.abs() + dx_err)
    if gate is not None:
        dg = scale * _to(n * t, gate.shape)
        out["gate"] = (dg, u * dg.abs() + abs(scale) * _to(n.abs() * (err + (64 + rows + x.shape[-1]) * E * big), gate.shape))
    return out


def _close(got, want, name):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    # (subnormal results are off by up to half their own step)
    tiny = {torch.float16: 2.0 ** -25}.get(name[1], 1e-38)
    bad = (got - value).abs() > bound + tiny
    assert not bad.any(), (name, int(bad.sum()), ((got - value).abs() / (bound + tiny)).max().item())


def _check(lead, k, dtype, stream, post, gate, scale, pre=True, seed=0):
    from primus_amd.pytorch import ops

    dev = torch.device("cuda:0")
    v, dy, dh = _inputs(lead, k, dtype, stream, post or not pre, gate, seed)
    want = _reference(v, dy if pre else None, dh, scale, dtype, stream, pre)
    v = {n: None if t is None else t.to(dev).requires_grad_() for n, t in v.items()}
    if pre:
        made = list(ops.add_rmsnorm(v["x"], v["residual"], v["weight"], EPS, post_weight=v["post_weight"], post_eps=POST_EPS, gate=v["gate"], scale=scale))
        given = [dy.to(dev), dh.to(dev)]
    else:
        v["weight"] = None
        made = [ops.rmsnorm_add(v["x"], v["residual"], v["post_weight"], POST_EPS, gate=v["gate"], scale=scale)]
        given = [dh.to(dev)]
    assert made[-1].dtype == stream and made[0].dtype == (dtype if pre else stream) and all(m.shape == v["x"].shape for m in made)
    names = [n for n, t in v.items() if t is not None]
    grads = dict(zip(names, torch.autograd.grad(made, [v[n] for n in names], given)))
    for name, got in list(zip(["y", "h"] if pre else ["h"], made)) + list(grads.items()):
        _close(got, want[name], (name, got.dtype))
        if name in grads:
            assert got.dtype == v[name].dtype


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
TYPES = [(BF, BF), (BF, FP), (HF, HF), (HF, FP), (FP, FP)]
# one row and one column; widths around the lanes' eights and the waves' sixty-fours; both kernels (256 and above) and both numbers of chunks (8192)
WIDTHS = [1, 7, 8, 9, 64, 65, 128, 129, 255, 256, 257, 512, 520, 1601, 4096, 8192, 8193, 16383, 16384]


@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("dtype,stream", TYPES)
def test_widths(gpu, k, dtype, stream):
    _check((5, 3), k, dtype, stream, False, "", 1.0)
    _check((3, 2), k, dtype, stream, True, "full", 0.5)
    _check((4, 3), k, dtype, stream, True, "column", -1.25, pre=False)


@pytest.mark.parametrize("gate", ["", "column", "element", "scalar", "first", "last", "token", "full", "first_scalar"])
@pytest.mark.parametrize("post,pre", [(False, True), (True, True), (True, False)])
@pytest.mark.parametrize("k", [40, 333, 1024])
def test_gates(gpu, gate, post, pre, k):
    for lead in ((1, 1), (2, 33), (67, 2), (3, 5, 7)):
        _check(lead, k, BF, FP, post, gate, 0.75, pre)
        _check(lead, k, HF, HF, post, gate, 1.0, pre)


@pytest.mark.parametrize("rows,k", [(1, 4096), (2, 2880), (700, 2880), (5000, 96), (40000, 8), (3001, 257), (530, 7168), (300, 12289)])
def test_rows(gpu, rows, k):
    _check((rows,), k, BF, BF, False, "", 1.0)
    _check((rows,), k, BF, FP, True, "token", 2.0)
    _check((rows,), k, FP, FP, True, "column", 1.0, pre=False)


@pytest.mark.parametrize("batch,seq,k", [(1500, 3, 512), (9000, 2, 64), (700, 1, 4096), (3, 2000, 512)])
def test_many_gates(gpu, batch, seq, k):
    """More gates than workers, and a few workers a gate; rows of a gate one after the other, or apart."""
    for gate in ("first", "last", "first_scalar"):
        _check((batch, seq), k, BF, BF, True, gate, 1.0)
        _check((seq, batch), k, HF, HF, False, gate, 1.0)


def test_one_dimension(gpu):
    from primus_amd.pytorch import ops

    x, r, w = (torch.randn(96, device=gpu) for _ in range(3))
    y, h = ops.add_rmsnorm(x, r, w)
    y2, h2 = ops.add_rmsnorm(x[None], r[None], w)
    assert y.shape == (96,) and torch.equal(y, y2[0]) and torch.equal(h, h2[0])


def test_no_rows(gpu):
    from primus_amd.pytorch import ops

    for shape, gate in (((0, 64), (64,)), ((0, 4, 640), (0, 1, 640)), ((2, 0, 64), (2, 1, 1))):
        x, r = (torch.empty(*shape, dtype=BF, device=gpu, requires_grad=True) for _ in range(2))
        w, p = (torch.ones(shape[-1], dtype=BF, device=gpu, requires_grad=True) for _ in range(2))
        g = torch.ones(*gate, dtype=BF, device=gpu, requires_grad=True)
        y, h = ops.add_rmsnorm(x, r, w, post_weight=p, gate=g)
        (y.sum() + h.sum()).backward()
        assert y.shape == h.shape == x.shape and x.grad.shape == x.shape
        assert not w.grad.any() and not p.grad.any() and not g.grad.any() and g.grad.shape == g.shape
        h = ops.rmsnorm_add(x, r, w, gate=g)
        assert h.shape == x.shape


def test_zero_rows_and_eps(gpu):
    """A row of zeros: y = 0, and with eps 0 what the formula has, 0 * inf."""
    from primus_amd.pytorch import ops

    x = torch.randn(4, 300, dtype=BF, device=gpu)
    x[1] = 0
    r = torch.zeros_like(x)
    w = torch.ones(300, dtype=BF, device=gpu)
    y, h = ops.add_rmsnorm(x, r, w, 1e-6)
    assert not y[1].any() and torch.equal(h, x) and torch.isfinite(y).all()
    y, _ = ops.add_rmsnorm(x, r, w, 0.0)
    assert y[1].isnan().all() and torch.isfinite(y[[0, 2, 3]]).all()


def test_what_is_not_finite_stays_in_its_row(gpu):
    from primus_amd.pytorch import ops

    for k in (40, 333, 9000):
        v, dy, dh = _inputs((6,), k, BF, BF, True, "token", device=gpu)
        bad = {n: None if t is None else t.clone() for n, t in v.items()}
        bad["x"][1, 3], bad["residual"][2, k - 1], bad["gate"][4, 0] = math.inf, math.nan, math.inf
        run = lambda a: ops.add_rmsnorm(a["x"], a["residual"], a["weight"], EPS, post_weight=a["post_weight"], gate=a["gate"])  # noqa: E731
        keep = [0, 3, 5]
        made, want = [], []
        for a, to in ((bad, made), (v, want)):
            a = {n: t.clone().requires_grad_() for n, t in a.items()}
            y, h = run(a)
            to += [y, h, *torch.autograd.grad([y, h], [a["x"], a["residual"], a["gate"]], [dy, dh])]
        for got, ref in zip(made, want):
            assert torch.equal(got[keep], ref[keep])
            assert not torch.isfinite(got[2]).all()
        assert not torch.isfinite(made[0][1]).all() and not torch.isfinite(made[1][4]).all()


def test_strides_offsets_and_orders(gpu):
    """Tensors that are not contiguous, or begin at an odd element: the same bits as their copies."""
    from primus_amd.pytorch import ops

    g = torch.Generator(device=gpu).manual_seed(5)
    for k in (24, 333, 1024):
        wide = torch.randn(4, 6, 2 * k + 1, generator=g, device=gpu).to(BF)
        x, r = wide[:, ::2, 1:k + 1], wide[:, ::2, k + 1:].transpose(0, 1).contiguous().transpose(0, 1)
        buf = torch.randn(k * 3 + 7, generator=g, device=gpu).to(BF)
        w, p, gate = buf[1:k + 1], buf[k + 3:2 * k + 3], buf[2 * k + 5:3 * k + 5].view(1, 1, k)
        odd = torch.empty(12 * k + 1, dtype=BF, device=gpu)[1:].view(4, 3, k)
        odd.copy_(x)
        out = []
        for a in ((x, r, w, p, gate), tuple(t.clone(memory_format=torch.contiguous_format) for t in (x, r, w, p, gate)), (odd, r, w, p, gate)):
            a = [t.detach().requires_grad_() for t in a]
            y, h = ops.add_rmsnorm(a[0], a[1], a[2], post_weight=a[3], gate=a[4], scale=0.5)
            gy, gh = (torch.ones(3, 4, k, dtype=BF, device=gpu).transpose(0, 1) * s for s in (1.0, 0.5))
            out.append([y, h, *torch.autograd.grad([y, h], a, [gy, gh])])
        for got in out[1:]:
            assert all(torch.equal(a, b) for a, b in zip(got, out[0]))


def test_gradients_that_are_not_asked_for(gpu):
    from primus_amd.pytorch import ops

    for k, gate, has_post in ((64, "first", True), (600, "first", True), (64, "token", True), (600, "token", True), (600, "token", False), (9000, "token", False),
                              (600, "column", False), (9001, "element", True)):
        v, dy, dh = _inputs((5, 4), k, BF, FP, has_post, gate, device=gpu)
        v = {n: t for n, t in v.items() if t is not None}
        names = list(v)

        def grads(needed, pre=True, given=(True, True)):
            a = {n: t.detach().clone().requires_grad_(n in needed) for n, t in v.items() if t is not None}
            if pre:
                made = ops.add_rmsnorm(a["x"], a["residual"], a["weight"], EPS, post_weight=a.get("post_weight"), gate=a["gate"], scale=0.5)
            else:
                made = (ops.rmsnorm_add(a["x"], a["residual"], a["post_weight"], EPS, gate=a["gate"], scale=0.5),)
            use = [(m, d) for m, d, w in zip(made, (dy, dh) if pre else (dh,), given) if w]
            return dict(zip(needed, torch.autograd.grad([m for m, _ in use], [a[n] for n in needed], [d for _, d in use], allow_unused=True)))

        every = grads(names)
        for n in names:
            assert torch.equal(grads([n])[n], every[n]), n
        if has_post:
            post = [n for n in names if n != "weight"]
            every = grads(post, False)
            for n in post:
                assert torch.equal(grads([n], False)[n], every[n]), n
            assert torch.equal(every["residual"], dh)
        v["post_weight"] = v.get("post_weight")
        # y or h alone
        want = _reference(v, dy, None, 0.5, BF, FP, post_eps=EPS)
        for n, got in grads(names, given=(True, False)).items():
            _close(got, want[n], (n, got.dtype))
        want = _reference(v, None, dh, 0.5, BF, FP, post_eps=EPS)
        for n, got in grads(names, given=(False, True)).items():
            if n == "weight":
                assert not got.any()
            else:
                _close(got, want[n], (n, got.dtype))


def test_without_gradients(gpu):
    from primus_amd.pytorch import ops

    v, _, _ = _inputs((5, 4), 96, BF, BF, True, "", device=gpu)
    a = {n: None if t is None else t.requires_grad_() for n, t in v.items()}
    y, h = ops.add_rmsnorm(a["x"], a["residual"], a["weight"], post_weight=a["post_weight"])
    with torch.no_grad():
        y2, h2 = ops.add_rmsnorm(a["x"], a["residual"], a["weight"], post_weight=a["post_weight"])
    with torch.inference_mode():
        y3, h3 = ops.add_rmsnorm(a["x"], a["residual"], a["weight"], post_weight=a["post_weight"])
    assert y.requires_grad and not y2.requires_grad
    assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(y, y3) and torch.equal(h, h3)


def test_second_derivatives_raise(gpu):
    from primus_amd.pytorch import ops

    x, r, w = (torch.randn(*s, device=gpu, requires_grad=True) for s in ((3, 16), (3, 16), (16,)))
    y, h = ops.add_rmsnorm(x, r, w)
    (dx,) = torch.autograd.grad(y.sum() + h.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        dx.sum().backward()


def test_differences(gpu):
    """The gradients against central differences: those of the kernels' float32 outputs within rounding of the float64 formula's, whose distance from the
    gradient goes with the square of the step."""
    from primus_amd.pytorch import ops

    k, lead, scale = 129, (3, 5), 0.7
    v, dy, dh = _inputs(lead, k, FP, FP, True, "first", seed=3)
    g = torch.Generator().manual_seed(9)
    names = list(v)
    way = {n: torch.randn(t.shape, generator=g).double() / math.sqrt(t.numel()) for n, t in v.items()}

    def loss64(a):
        out = _reference(a, None, None, scale, FP, FP)
        return out["y"][0], out["h"][0]

    def at(n, step, kernels):
        a = {m: t.double() for m, t in v.items()}
        a[n] = a[n] + step * way[n]
        if kernels:
            a = {m: t.float() for m, t in a.items()}
            y, h = ops.add_rmsnorm(*(a[m].to(gpu) for m in ("x", "residual", "weight")), EPS, post_weight=a["post_weight"].to(gpu), post_eps=POST_EPS,
                                   gate=a["gate"].to(gpu), scale=scale)
            y, h = y.cpu().double(), h.cpu().double()
        else:
            y, h = loss64(a)
        return (y * dy.double()).sum() + (h * dh.double()).sum(), (y * dy.double()).abs().sum() + (h * dh.double()).abs().sum()

    a = {n: t.to(gpu).requires_grad_() for n, t in v.items()}
    made = ops.add_rmsnorm(a["x"], a["residual"], a["weight"], EPS, post_weight=a["post_weight"], post_eps=POST_EPS, gate=a["gate"], scale=scale)
    grads = dict(zip(names, torch.autograd.grad(made, [a[n] for n in names], [dy.to(gpu), dh.to(gpu)])))
    step = 2.0 ** -6
    for n in names:
        d64 = [((at(n, s, False)[0] - at(n, -s, False)[0]) / (2 * s)).item() for s in (step, 2 * step)]
        plus, minus = at(n, step, True), at(n, -step, True)
        d32 = ((plus[0] - minus[0]) / (2 * step)).item()
        # outputs within 64 e of what they are added up of, inputs rounded to fp32 once more
        rounding = 200 * E * (plus[1] + minus[1]).item() / (2 * step)
        assert abs(d32 - d64[0]) <= rounding, n
        slope = (grads[n].cpu().double() * way[n]).sum().item()
        # the difference at twice the step is four times as far off: a third of their distance, doubled for the higher terms; and the gradient's own rounding
        assert abs(slope - d64[0]) <= abs(d64[1] - d64[0]) + 200 * E * (plus[1]).item(), n


def test_same_bits_each_time(gpu):
    from primus_amd.pytorch import ops

    for lead, k, gate in (((300, 7), 96, "column"), ((3, 500), 2880, "first"), ((2, 300), 10000, "token")):
        v, dy, dh = _inputs(lead, k, BF, BF, True, gate, device=gpu)
        v = {n: t.requires_grad_() for n, t in v.items()}
        runs = []
        for _ in range(2):
            y, h = ops.add_rmsnorm(v["x"], v["residual"], v["weight"], post_weight=v["post_weight"], gate=v["gate"])
            runs.append([y, h, *torch.autograd.grad([y, h], list(v.values()), [dy, dh])])
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_rows_beyond_32_bit_offsets(gpu):
    """More than 2^31 elements: the last rows are those of a call on them alone."""
    from primus_amd.pytorch import ops

    k, rows = 16384, (1 << 17) + 24
    x = torch.zeros(rows, k, dtype=BF, device=gpu)
    r = torch.zeros(rows, k, dtype=BF, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    x[-40:] = torch.randn(40, k, generator=g, device=gpu).to(BF)
    r[-40:] = torch.randn(40, k, generator=g, device=gpu).to(BF)
    w = torch.randn(k, generator=g, device=gpu).to(BF).requires_grad_()
    x.requires_grad_()
    y, h = ops.add_rmsnorm(x, r, w)
    dy = torch.zeros_like(h)
    dy[-40:] = torch.randn(40, k, generator=g, device=gpu).to(BF)
    dx, = torch.autograd.grad(y, x, dy)
    xs = x.detach()[-40:].clone().requires_grad_()
    ys, hs = ops.add_rmsnorm(xs, r[-40:], w)
    dxs, = torch.autograd.grad(ys, xs, dy[-40:].clone())
    assert torch.equal(y[-40:], ys) and torch.equal(h[-40:], hs) and torch.equal(dx[-40:], dxs)
    assert not y[:-40].any() and not dx[:-40].any()


@pytest.mark.parametrize("k,rows", [(64, (1 << 23) + 100), (1, (1 << 29) + (1 << 20)), (4, (1 << 28) + 40)])
def test_many_short_rows(gpu, k, rows):
    """Short rows whose tensor passes the descriptors' offsets, and more of them than a launch has threads for: the last rows are those of a
    call on them alone, forward and backward."""
    from primus_amd.pytorch import ops

    x, r = (torch.zeros(rows, k, dtype=BF, device=gpu) for _ in range(2))
    g = torch.Generator(device=gpu).manual_seed(1)
    x[-70:], r[-70:] = (torch.randn(70, k, generator=g, device=gpu).to(BF) for _ in range(2))
    w = torch.randn(k, generator=g, device=gpu).to(BF)
    dy = torch.zeros(rows, k, dtype=BF, device=gpu)
    dy[-70:] = torch.randn(70, k, generator=g, device=gpu).to(BF)
    out = []
    for a in ((x, r, dy), tuple(t[-70:].clone() for t in (x, r, dy))):
        xs = a[0].requires_grad_()
        y, h = ops.add_rmsnorm(xs, a[1], w)
        (dx,) = torch.autograd.grad(y, xs, a[2])
        out.append([t[-70:].clone() for t in (y, h, dx)])
        if len(y) > 70:
            assert not y[:-70].any() and not dx[:-70].any()
        del y, h, dx
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_one_tensor_twice(gpu):
    """x and the residual one tensor, a weight used by both norms, a gradient handed to several inputs."""
    from primus_amd.pytorch import ops

    for k in (64, 700):
        g = torch.Generator().manual_seed(k)
        x, w, dy, dh = (torch.randn(s, generator=g) for s in ((6, k), (k,), (6, k), (6, k)))
        a, b = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
        y, h = ops.add_rmsnorm(a, a, b, EPS)
        got = torch.autograd.grad([y, h], [a, b], [dy.to(gpu), dh.to(gpu)])
        want = _reference(dict(x=x, residual=x, weight=w, post_weight=None, gate=None), dy, dh, 1.0, FP, FP)
        _close(got[0], (2 * want["x"][0], 2 * want["x"][1]), ("x twice", FP))
        _close(got[1], want["weight"], ("weight", FP))
        y, h = ops.add_rmsnorm(a, a, b, EPS, post_weight=b, post_eps=POST_EPS)
        got = torch.autograd.grad([y, h], [a, b], [dy.to(gpu), dh.to(gpu)])
        want = _reference(dict(x=x, residual=x, weight=w, post_weight=w, gate=None), dy, dh, 1.0, FP, FP)
        for g1, n1, n2 in ((got[0], "x", "residual"), (got[1], "weight", "post_weight")):
            # (and the sum of the two, half a step)
            _close(g1, (want[n1][0] + want[n2][0], want[n1][1] + want[n2][1] + E * (want[n1][0] + want[n2][0]).abs()), (n1, FP))


def test_saved_tensors_that_come_back_otherwise_are_refused(gpu):
    from primus_amd.pytorch import ops

    v, dy, dh = _inputs((4, 4), 96, BF, BF, True, "", device=gpu)
    v = {n: t.requires_grad_() for n, t in v.items() if t is not None}
    for pack, unpack in ((lambda t: t, lambda t: t.transpose(0, 1) if t.dim() > 1 else t), (lambda t: t, lambda t: t.float() if t.dtype == BF else t.double()),
                         (lambda t: t, lambda t: t[:1])):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            made = ops.add_rmsnorm(v["x"], v["residual"], v["weight"], post_weight=v["post_weight"])
        with pytest.raises(ValueError, match="contiguous"):
            torch.autograd.grad(made, list(v.values()), [dy, dh])


@pytest.mark.parametrize("k", [640, 9000])
def test_on_another_stream_and_captured(gpu, k):
    """On a side stream, and in a graph replayed on new inputs with eager work between the replays."""
    from primus_amd.pytorch import ops

    v, dy, dh = _inputs((4, 50), k, BF, FP, True, "first", device=gpu)
    names = list(v)

    def run(a, dy, dh):
        a = {n: t.detach().requires_grad_() for n, t in a.items()}
        y, h = ops.add_rmsnorm(a["x"], a["residual"], a["weight"], EPS, post_weight=a["post_weight"], gate=a["gate"], scale=0.5)
        z = ops.rmsnorm_add(y, h, a["post_weight"], EPS, gate=a["gate"])
        return [y.detach(), h.detach(), z.detach(), *torch.autograd.grad([z, h], list(a.values()), [dh, dh])]

    want = run(v, dy, dh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(v, dy, dh)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = {n: t.clone() for n, t in v.items()}
    sdy, sdh = dy.clone(), dh.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(static, sdy, sdh)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static, sdy, sdh)
    for seed in range(4):
        new, ndy, ndh = _inputs((4, 50), k, BF, FP, True, "first", seed=seed, device=gpu)
        for n in names:
            static[n].copy_(new[n])
        sdy.copy_(ndy), sdh.copy_(ndh)
        graph.replay()
        torch.cuda.synchronize()
        want = run(new, ndy, ndh)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_through_host_memory(gpu):
    from primus_amd.pytorch import ops

    v, dy, dh = _inputs((4, 5), 96, BF, BF, True, "token", device=gpu)
    v = {n: t.requires_grad_() for n, t in v.items()}
    run = lambda: ops.add_rmsnorm(v["x"], v["residual"], v["weight"], post_weight=v["post_weight"], gate=v["gate"])  # noqa: E731
    want = torch.autograd.grad(run(), list(v.values()), [dy, dh])
    with torch.autograd.graph.save_on_cpu():
        made = run()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(made, list(v.values()), [dy, dh]), want))


def test_rows_around_the_output_stay(gpu):
    """The C ABI on views of larger buffers: what is before and behind the rows is not touched."""
    from primus_amd import _lib
    from primus_amd.pytorch import kernels as K

    lib = _lib.load()
    for rows, k, dt in ((3, 33, BF), (5, 700, HF), (2, 8200, FP)):
        n = rows * k
        bufs = [torch.full((n + 18,), 7.0, dtype=dt, device=gpu) for _ in range(2)]
        y, h = (b[9:9 + n].view(rows, k) for b in bufs)
        x, r = torch.randn(rows, k, device=gpu).to(dt), torch.randn(rows, k, device=gpu).to(dt)
        w = torch.randn(k, device=gpu).to(dt)
        rc = lib.mxl_block_norm(x.data_ptr(), r.data_ptr(), rows, k, K._DT[dt], K._DT[dt], None, 0.0, None, 1, 1, 0, 1.0, w.data_ptr(), EPS, y.data_ptr(), h.data_ptr(),
                                None, None, K._stream())
        assert rc == 0
        wy, wh, _, _ = K.block_norm_impl(x, r, w, EPS, None, 0.0, None, 1.0)
        assert torch.equal(y, wy) and torch.equal(h, wh)
        assert all((b[:9] == 7).all() and (b[9 + n:] == 7).all() for b in bufs)


@pytest.mark.parametrize("k", [40, 333, 1024, 9000])
def test_an_infinite_gate_leaves_its_own_sums(gpu, k):
    """An element of a gate that is infinite: the post weight's gradient is infinite in its column, as the formula's is, and the other columns' finite."""
    from primus_amd.pytorch import ops

    rows, column = 6, 3
    for dtype, stream in ((BF, FP), (HF, HF)):
        v, _, dh = _inputs((rows,), k, dtype, stream, True, "full", device=gpu)
        for row in (0, rows - 1):
            gate = v["gate"].clone()
            gate[row, column] = math.inf
            wp = v["post_weight"].clone().requires_grad_()
            (got,) = torch.autograd.grad(ops.rmsnorm_add(v["x"], v["residual"], wp, POST_EPS, gate=gate), wp, dh)
            want = math.copysign(math.inf, (dh[row, column].double() * v["x"][row, column].double()).item())
            assert got[column].item() == want, (dtype, row)
            rest = [c for c in range(k) if c != column]
            assert torch.isfinite(got[rest]).all()


@pytest.fixture()
def released():
    """Large tensors go back to the device: a later test of memory held may be given one of their blocks, which count whole."""
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _signs(shape, g, dtype, device):
    return (2 * torch.randint(0, 2, shape, generator=g) - 1).to(dtype).to(device)


def _few(rows, k, g):
    """[rows, k] of -1, 0 and 1, something in every row, and about 2500 (at least rows / k) a column, 2500 a row, that are not 0: sums stay below 256."""
    each = max(1, min(k, 2500 * k // rows, 2500))
    at = (torch.randint(0, k, (rows, 1), generator=g) + torch.arange(each) * (k // each)) % k
    return torch.zeros(rows, k).scatter_(1, at, _signs((rows, each), g, torch.float32, "cpu"))


@pytest.mark.parametrize("lead,k", [((40000,), 8), ((5000,), 96), ((9000, 2), 64), ((2, 9000), 64), ((3001,), 257), ((70, 43), 257), ((530,), 7168), ((300,), 12289), ((1500, 3), 512),
                                    ((33, 31), 129), ((1023,), 1601)])
@pytest.mark.parametrize("gate", ["", "column", "first", "last", "token", "full"])
def test_every_row_counts(gpu, released, lead, k, gate):
    """Sums over rows that are whole numbers: a row, a worker or a wave that is left out changes them by one at least.  x and gate are 1 or -1, so a row's
    normalised values are too, but for the rounding of 1 / k and of the root: below 2^-22 in all, rows * 2^-22 in a sum, which is under 1 / 4.  Whole numbers
    up to 256 are a bf16's, and what is so close to one rounds to it."""
    from primus_amd.pytorch import ops

    rows = math.prod(lead)
    g = torch.Generator().manual_seed(k + rows)
    one = torch.ones(k)
    whole = lambda t, w, name: _whole(t, w, name + (gate,))  # noqa: E731
    for dtype, stream in ((BF, BF), (HF, FP), (FP, FP)):
        x = _signs(lead + (k,), g, dtype, gpu)
        shape = _gate_shape(gate, lead, k)
        a = {"x": x, "residual": torch.zeros(lead + (k,), dtype=stream, device=gpu), "weight": one.to(dtype).to(gpu), "post_weight": one.to(dtype).to(gpu),
             "gate": None if shape is None else _signs(shape, g, dtype, gpu)}
        d = _few(rows, k, g).view(lead + (k,))
        n = x.cpu().float() * d
        f = n if shape is None else n * a["gate"].cpu().float()
        want = {"weight": f.reshape(rows, k).sum(0), "post_weight": f.reshape(rows, k).sum(0), "gate": None if shape is None else _to(n, shape)}
        assert want["weight"].abs().max() <= 256 and (shape is None or want["gate"].abs().max() <= 256)     # (of the data, by its seed)
        a = {name: None if t is None else t.requires_grad_() for name, t in a.items()}
        for post in (False, True):
            y, h = ops.add_rmsnorm(a["x"], a["residual"], a["weight"], 0.0, post_weight=a["post_weight"] if post else None, gate=a["gate"])
            (dw,) = torch.autograd.grad(y, a["weight"], d.to(dtype).to(gpu), retain_graph=True)
            whole(dw, want["weight"], ("weight", post, dtype))
            names = [m for m in ("post_weight", "gate") if (post or m == "gate") and a[m] is not None]
            if names:
                for m, got in zip(names, torch.autograd.grad(h, [a[m] for m in names], d.to(stream).to(gpu))):
                    whole(got, want[m], (m, post, dtype))
        h = ops.rmsnorm_add(a["x"], a["residual"], a["post_weight"], 0.0, gate=a["gate"])
        names = [m for m in ("post_weight", "gate") if a[m] is not None]
        for m, got in zip(names, torch.autograd.grad(h, [a[m] for m in names], d.to(stream).to(gpu))):
            whole(got, want[m], (m, "alone", dtype))


def _whole(got, want, name):
    off = (got.detach().cpu().float() - want).abs()
    assert got.shape == want.shape and (off <= 0.25).all(), (name, int((off > 0.25).sum()), off.max().item())


@pytest.mark.parametrize("k,rows", [(16384, (1 << 17) + 24), (64, (1 << 23) + 100), (4, (1 << 28) + 40)])
def test_weight_gradients_beyond_32_bit_offsets(gpu, released, k, rows):
    """The weights' gradients of more rows than 31 bits of offsets reach, of which the first, the last and some between are not zero: whole numbers, as above."""
    from primus_amd.pytorch import ops

    g = torch.Generator().manual_seed(k)
    at = sorted({0, 1, rows // 2, rows - 65, *range(rows - 40, rows)} | set(torch.randint(0, rows, (60,), generator=g).tolist()))
    x, dy = (torch.zeros(rows, k, dtype=BF, device=gpu) for _ in range(2))
    r = torch.zeros(rows, k, dtype=BF, device=gpu)
    sx, sd = (_signs((len(at), k), g, BF, gpu) for _ in range(2))
    where = torch.tensor(at, device=gpu)
    x[where], dy[where] = sx, sd
    want = (sx.float() * sd.float()).sum(0).cpu()
    w = torch.ones(k, dtype=BF, device=gpu, requires_grad=True)
    y, h = ops.add_rmsnorm(x, r, w, 1e-6)       # (1 / sqrt(1 + 1e-6): 1e-6 * 110 rows off)
    (dw,) = torch.autograd.grad(y, w, dy)
    _whole(dw, want, ("weight", k))
    del y, h
    h = ops.rmsnorm_add(x, r, w, 1e-6)
    (dw,) = torch.autograd.grad(h, w, dy)
    _whole(dw, want, ("post_weight", k))


@pytest.mark.parametrize("k", [40, 333, 1024, 9000])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_weight_gradient_of_the_sums_before_their_rounding(gpu, dtype, k):
    """With a stream of 16 bits dweight = sum dy * hh has hh of the sums that y was made of, not of h as it was rounded.  hh is off by the fp32 work on what
    is added up in h, 64 e of its magnitudes; then the bars of the sum and of its one rounding."""
    from primus_amd.pytorch import ops

    for lead, post, gate, scale in (((3, 67), False, "", 1.0), ((201,), False, "", -0.75), ((3, 67), True, "", 0.5), ((3, 67), True, "first", 1.0), ((67, 3), False, "last", 1.0),
                                    ((201,), True, "token", 1.0), ((3, 67), False, "full", 1.25), ((201,), False, "element", 1.0)):
        v, dy, _ = _inputs(lead, k, dtype, dtype, post, gate)
        d = {n: None if t is None else t.double() for n, t in v.items()}
        x = d["x"] if not post else d["x"] / torch.sqrt((d["x"] ** 2).mean(-1, keepdim=True) + POST_EPS) * d["post_weight"]
        add = scale * x * (1 if d["gate"] is None else d["gate"])
        h = d["residual"] + add
        r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
        rows = math.prod(lead)
        total = lambda t: t.reshape(rows, k).sum(0)  # noqa: E731
        want = total(dy.double() * h * r)
        bar = _u(dtype) * want.abs() + total(dy.double().abs() * (64 * E * (d["residual"].abs() + add.abs()) * r + (64 + rows) * E * (h * r).abs()))
        a = {n: None if t is None else t.to(gpu).requires_grad_() for n, t in v.items()}
        for wanted in ([n for n in a if a[n] is not None], ["weight"]):
            y, _ = ops.add_rmsnorm(a["x"], a["residual"], a["weight"], EPS, post_weight=a["post_weight"], post_eps=POST_EPS, gate=a["gate"], scale=scale)
            got = torch.autograd.grad(y, [a[n] for n in wanted], dy.to(gpu))[wanted.index("weight")]
            _close(got, (want, bar), ("weight", dtype))
