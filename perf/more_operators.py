"""What stands at the ends of a training step's blocks and after its backward, as cases that can be timed and compared: the norm
before a block with the residual add in front of it (``ops.add_rmsnorm``, also with the norm after the previous block, its gate
and its residual scale), the norm after a block (``ops.rmsnorm_add``), the global norm of many gradients (``ops.grad_norm``) and
their clipping (``ops.clip_grads``).

``own`` False: every operator in its plain form, elementary torch operations in 32 bits (long sums in 64); True: the calls a
program makes of the framework.

A case holds ``op`` and the operator's sizes and options; ``backward``: the pass takes the gradients too.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- the cases ----------------------------------------------------------------------------------------------------
def _norm(name, op, batch, seq, hidden, dtype="bf16", stream="", post=False, gate="", scale=1.0, backward=True):
    """``stream``: type of the residual stream if it is not ``dtype``; ``gate``: "column" [hidden], "batch" [batch, 1, hidden],
    "token" [batch, seq, 1], "full" [batch, seq, hidden] or none; ``post``: the norm after the previous block too."""
    return dict(name=name, op=op, batch=batch, seq=seq, hidden=hidden, dtype=dtype, stream=stream or dtype, post=post, gate=gate, scale=scale,
                backward=backward)


def _grads(name, op, shapes, dtype="fp32", kind="2", out="", limit=0.25):
    """``shapes``: "28672x4096 2*4096" is one matrix and two vectors; ``kind``: "2" or "max"; ``out``: type of the tensors that the
    clipped gradients go to (none: in place); ``limit``: the largest norm allowed, in units of about what the inputs have."""
    return dict(name=name, op=op, shapes=shapes, dtype=dtype, kind=kind, out=out, limit=limit)


# a layer of Llama-3-8B: attention's two projections, the MLP's two and the norms
_LLAMA_LAYER = "6144x4096 4096x4096 28672x4096 4096x14336 2*4096"


def listed():
    return [
        # a decode step of 8 sequences at Llama-3-8B's width
        _norm("prenorm_decode", "prenorm", 8, 1, 4096, backward=False),
        # Mixtral-8x7B training: residual add and norm of 16384 tokens
        _norm("prenorm_train", "prenorm", 4, 4096, 4096),
        # norms on both sides of the blocks at GPT-OSS's width, odd length, gate a sequence, the stream kept in fp32
        _norm("prenorm_sandwich", "prenorm", 3, 1801, 2880, stream="fp32", post=True, gate="batch", scale=0.5),
        # a width that is no multiple of anything
        _norm("prenorm_odd", "prenorm", 2, 777, 1601, dtype="fp16", gate="full"),
        # a decode step of one token at DeepSeek-V3's width
        _norm("postnorm_decode", "postnorm", 1, 1, 7168, backward=False),
        # DeepSeek-V3 width, 8192 tokens, a learned factor a channel
        _norm("postnorm_train", "postnorm", 2, 4096, 7168, gate="column"),
        # a short batch whose tokens have a gate each
        _norm("postnorm_short", "postnorm", 1, 333, 2880, dtype="fp16", gate="token", scale=1.25),
        # many small tensors: norms and biases of a deep model
        _grads("norm_small", "norm", "64*4096 32*6144 64*2880 32*128 33*1601", dtype="bf16"),
        # the main gradients of a Mixtral-8x7B layer's experts
        _grads("norm_experts", "norm", "8x28672x4096 8x4096x14336 8x4096"),
        # the largest gradient of a Llama-3-8B layer
        _grads("norm_max", "norm", _LLAMA_LAYER, dtype="bf16", kind="max"),
        # bf16 gradients of a Llama-3-8B layer, clipped into the optimizer's fp32 ones
        _grads("clip_layer", "clip", _LLAMA_LAYER, dtype="bf16", out="fp32"),
        # the same layer's main gradients within the bound
        _grads("clip_within", "clip", _LLAMA_LAYER, limit=4.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("prenorm", "prenorm", "postnorm", "norm", "clip"))
    if op in ("prenorm", "postnorm"):
        hidden = _log(rng, 64, 16384) if rng.random() < 0.3 else 32 * _log(rng, 2, 512)
        tokens = _log(rng, 1, max(1, (1 << 25) // hidden))
        batch = rng.choice((1, 2, 3, 4, 8))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        c = _norm("", op, batch, max(1, tokens // batch), hidden, dtype=dtype, stream=rng.choice(("", "fp32")), post=op == "prenorm" and rng.random() < 0.5,
                  gate=rng.choice(("", "", "column", "batch", "token", "full")), scale=rng.choice((1.0, 0.5, 1.25)), backward=rng.random() < 0.7)
    else:
        count = _log(rng, 1, 200)
        total = _log(rng, 256, 1 << 28)
        parts = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(count)]
        sizes = [max(1, int(total * p / sum(parts))) for p in parts]
        c = _grads("", op, " ".join(str(n) for n in sizes), dtype=rng.choice(("fp32", "bf16", "fp16", "mixed")), kind=rng.choice(("2", "2", "max")),
                   out=rng.choice(("fp32", "bf16")) if op == "clip" else "", limit=rng.choice((0.25, 0.25, 4.0)))
    del c["name"]
    return c


# ---- inputs -------------------------------------------------------------------------------------------------------
def _gate_shape(c):
    b, s, k = c["batch"], c["seq"], c["hidden"]
    return {"column": (k,), "batch": (b, 1, k), "token": (b, s, 1), "full": (b, s, k)}[c["gate"]]


def _shapes(c):
    out = []
    for part in c["shapes"].split():
        times, _, dims = part.rpartition("*")
        out += [tuple(int(d) for d in dims.split("x"))] * int(times or 1)
    return out


def _grad_dtype(c, i):
    return (torch.float32, torch.bfloat16, torch.float16)[i % 3] if c["dtype"] == "mixed" else _DTYPES[c["dtype"]]


_GRAD_SCALES = (1e-3, 3e-3, 1e-2)       # of the tensors in turn


def _max_norm(c):
    sizes = [math.prod(shape) for shape in _shapes(c)]
    if c["kind"] == "max":
        return c["limit"] * 5.0 * max(_GRAD_SCALES[:len(sizes)])
    return c["limit"] * math.sqrt(sum(n * _GRAD_SCALES[i % 3] ** 2 for i, n in enumerate(sizes)))


def _leaves(c):
    return ["x", "residual", "weight"] + (["post_weight"] if c["post"] else []) + (["gate"] if c["gate"] else [])


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    dev = gen.device
    s = {"case": c}

    def normal(*shape, dtype=torch.float32, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale + mean).to(dtype)

    if c["op"] in ("prenorm", "postnorm"):
        b, l, k = c["batch"], c["seq"], c["hidden"]
        dt, st = _DTYPES[c["dtype"]], _DTYPES[c["stream"]]
        s["x"], s["residual"] = normal(b, l, k, dtype=dt), normal(b, l, k, dtype=st, scale=2.0)
        s["weight"] = normal(k, dtype=dt, scale=0.1, mean=1.0)
        s["post_weight"] = normal(k, dtype=dt, scale=0.1, mean=1.0) if c["post"] else None
        s["gate"] = normal(*_gate_shape(c), dtype=dt, scale=0.5, mean=0.5) if c["gate"] else None
        if c["backward"]:
            s["dh"] = normal(b, l, k, dtype=st)
            s["dy"] = normal(b, l, k, dtype=dt) if c["op"] == "prenorm" else None
            for name in _leaves(c):
                s[name].requires_grad_(own)
    else:
        s["grads"] = [normal(*shape, dtype=_grad_dtype(c, i), scale=_GRAD_SCALES[i % 3]) for i, shape in enumerate(_shapes(c))]
        if c["op"] == "clip":
            s["max_norm"] = _max_norm(c)
            s["out"] = [torch.empty(g.shape, dtype=_DTYPES[c["out"]], device=dev) for g in s["grads"]] if c["out"] else None
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _rstd(v):
    return 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)


def _to_shape(t, shape):
    """``t`` summed over what ``shape`` broadcasts over."""
    dims = [d for d in range(t.dim()) if d < t.dim() - len(shape) or shape[d - t.dim() + len(shape)] == 1 != t.shape[d]]
    return (t.sum(dims) if dims else t).reshape(shape)


def _plain_norm(s):
    c = s["case"]
    dt, st = _DTYPES[c["dtype"]], _DTYPES[c["stream"]]
    pre = c["op"] == "prenorm"
    x, res = s["x"].float(), s["residual"].float()
    wp = s["post_weight"].float() if c["post"] else None if pre else s["weight"].float()
    n = x
    if wp is not None:
        rp = _rstd(x)
        xh = x * rp
        n = xh * wp
    factor = c["scale"] if s["gate"] is None else c["scale"] * s["gate"].float()
    h = res + factor * n
    out = [h.to(st)]
    if pre:
        r, w = _rstd(h), s["weight"].float()
        hh = h * r
        out = [(hh * w).to(dt)] + out
    if not c["backward"]:
        return out
    t = s["dh"].float()
    dw = None
    if pre:
        dy = s["dy"].float()
        g = dy * w
        t = t + r * (g - hh * (g * hh).mean(-1, keepdim=True))
        dw = (dy * hh).sum((0, 1))
    dn = factor * t
    dx, dwp = dn, None
    if wp is not None:
        dwp = (dn * xh).sum((0, 1))
        g = dn * wp
        dx = rp * (g - xh * (g * xh).mean(-1, keepdim=True))
    out += [dx.to(dt), t.to(st), (dw if pre else dwp).to(dt)]
    if c["post"]:
        out.append(dwp.to(dt))
    if s["gate"] is not None:
        out.append((c["scale"] * _to_shape(n * t, s["gate"].shape)).to(dt))
    return out


def _plain_total(c, grads):
    if c["kind"] == "max":
        return torch.stack([g.float().abs().max() for g in grads]).max()
    total = torch.zeros((), dtype=torch.float64, device=grads[0].device)
    for g in grads:
        f = g.float()
        total = total + (f * f).sum(dtype=torch.float64)
    return torch.sqrt(total).float()


def _plain_grads(s):
    c, grads = s["case"], s["grads"]
    norm = _plain_total(c, grads)
    if c["op"] == "norm":
        return [norm]
    coefficient = torch.clamp(s["max_norm"] / (norm.double() + 1e-6), max=1.0)
    targets = grads if s["out"] is None else s["out"]
    for g, o in zip(grads, targets):
        o.copy_(g * coefficient.float() if g.dtype == torch.float32 else g.float() * coefficient.float())
    return [norm] + targets


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _own_norm(s):
    from primus_amd.pytorch import ops

    c = s["case"]
    if c["op"] == "prenorm":
        made = list(ops.add_rmsnorm(s["x"], s["residual"], s["weight"], EPS, post_weight=s["post_weight"], gate=s["gate"], scale=c["scale"]))
        given = [s.get("dy"), s.get("dh")]
    else:
        made = [ops.rmsnorm_add(s["x"], s["residual"], s["weight"], EPS, gate=s["gate"], scale=c["scale"])]
        given = [s.get("dh")]
    out = [t.detach() for t in made]
    if c["backward"]:
        out += torch.autograd.grad(made, [s[name] for name in _leaves(c)], given)
    return out


def _own_grads(s):
    from primus_amd.pytorch import ops

    c = s["case"]
    kind = math.inf if c["kind"] == "max" else 2.0
    if c["op"] == "norm":
        return [ops.grad_norm(s["grads"], kind)]
    norm = ops.clip_grads(s["grads"], s["max_norm"], norm_type=kind, out=s["out"])
    return [norm] + (s["grads"] if s["out"] is None else s["out"])


def run(state):
    if state["case"]["op"] in ("prenorm", "postnorm"):
        return (_own_norm if own else _plain_norm)(state)
    return (_own_grads if own else _plain_grads)(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    c = case
    size = {"fp32": 4, "bf16": 2, "fp16": 2, "mixed": 8 / 3, "": 0}
    if c["op"] in ("prenorm", "postnorm"):
        n, k = c["batch"] * c["seq"] * c["hidden"], c["hidden"]
        e, st, pre = size[c["dtype"]], size[c["stream"]], c["op"] == "prenorm"
        gate = math.prod(_gate_shape(c)) if c["gate"] else 0
        weights = k * (2 if c["post"] else 1)
        nbytes = n * (e + 2 * st) + (n * e if pre else 0) + e * (weights + gate)
        flops = n * (12 if c["post"] else 8)
        if c["backward"]:
            # dh and dy in, the gradients of x and of the residual out (one tensor where they are the same, dh where it is the residual's)
            same = pre and not c["post"] and not c["gate"] and c["scale"] == 1.0 and c["stream"] == c["dtype"]
            nbytes += n * st + n * e + (n * e if pre else 0) + (n * st if pre and not same else 0) + e * (weights + gate)
            flops += n * (24 if c["post"] else 14)
        return {"bytes": int(nbytes), "flops": int(flops)}
    n = sum(math.prod(shape) for shape in _shapes(c))
    nbytes, flops = n * size[c["dtype"]] + 4, 2 * n
    if c["op"] == "clip":
        if c["out"] or c["limit"] < 1.0:
            nbytes += n * size[c["out"] or c["dtype"]]
            flops += n
    return {"bytes": int(nbytes), "flops": int(flops)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _exact_norm(s):
    """The formulas as torch's graph of 64-bit operations, its gradients by the graph."""
    c = s["case"]
    names = _leaves(c)
    v = {name: s[name].detach().double().requires_grad_(c["backward"]) for name in names}

    def rms(t, w):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * w

    if c["op"] == "postnorm":
        n = rms(v["x"], v["weight"])
    else:
        n = rms(v["x"], v["post_weight"]) if c["post"] else v["x"]
    if c["gate"]:
        n = n * v["gate"]
    h = v["residual"] + n * c["scale"]
    made, given = [h], [s.get("dh")]
    if c["op"] == "prenorm":
        made, given = [rms(h, v["weight"]), h], [s.get("dy"), s.get("dh")]
    out = [t.detach() for t in made]
    if c["backward"]:
        out += torch.autograd.grad(made, [v[name] for name in names], [g.double() for g in given])
    return out


def _exact_total(c, grads):
    pieces = [p for g in grads for p in torch.split(g.reshape(-1), 1 << 26)]
    if c["kind"] == "max":
        return max(max(abs(p.max().item()), abs(p.min().item())) for p in pieces)
    return math.sqrt(math.fsum(torch.dot(p.double(), p.double()).item() for p in pieces))


def _exact_grads(s):
    c = s["case"]
    norm = _exact_total(c, s["grads"])
    out = [torch.tensor(norm, dtype=torch.float64, device=s["grads"][0].device)]
    if c["op"] == "clip":
        factor = min(1.0, s["max_norm"] / (norm + 1e-6))
        out += [g.double() * factor for g in s["grads"]]
    return out


def exact(case, seed):
    """What ``run`` returns for these inputs, from the definitions in 64 bits."""
    global own
    was, own = own, False       # the inputs as they are, without a graph
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return (_exact_norm if case["op"] in ("prenorm", "postnorm") else _exact_grads)(s)
