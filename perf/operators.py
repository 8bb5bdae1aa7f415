"""Measured cases of the operators that train a deep KAN stack: the orthogonalised update of a weight matrix, the Muon
step of a model, and the group norm with an activation between two layers, on values and on derivative jets.

``run`` makes one pass: in elementary torch operations in 32 bits, or, where ``own`` is set, through this package.
"""
import math

import torch

own = False

#: the odd quintic of one Newton-Schulz step, x -> a x + b x^3 + c x^5 on the singular values
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_EPS, NORM_EPS = 1e-7, 1e-5
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # the base weight of the hidden layer of KAN [2, 64, 64, 1]: the smallest call, where launches count
        {"name": "orthogonalize 64x64 f32", "op": "orthogonalize", "batch": 1, "rows": 64, "cols": 64, "dtype": "float32"},
        # the spline weight of a hidden layer of KAN [2, 256, 256, 256, 1] at grid 20: 23 coefficients an edge
        {"name": "orthogonalize 256x5888 f32", "op": "orthogonalize", "batch": 1, "rows": 256, "cols": 5888,
         "dtype": "float32"},
        # a stack of tall weights of odd sizes in half precision
        {"name": "orthogonalize 4x1000x771 f16", "op": "orthogonalize", "batch": 4, "rows": 1000, "cols": 771,
         "dtype": "float16"},
        # a large matrix with gradients in bfloat16
        {"name": "orthogonalize 2048x8192 bf16", "op": "orthogonalize", "batch": 1, "rows": 2048, "cols": 8192,
         "dtype": "bfloat16"},
        # one optimiser step of KAN [2, 64, 64, 1], grid 10 (nine matrices, the largest 64 x 832)
        {"name": "muon KAN 2-64-64-1 grid 10", "op": "muon", "width": 64, "hidden": 2, "grid": 10},
        # one optimiser step of KAN [2, 256, 256, 256, 1], grid 20 (twelve matrices, the largest 256 x 5888)
        {"name": "muon KAN 2-256-256-256-1 grid 20", "op": "muon", "width": 256, "hidden": 3, "grid": 20},
        # evaluation of a trained stack on ten thousand points
        {"name": "norm 10000x64 f32 tanh", "op": "norm", "n": 10000, "s": 1, "channels": 64, "groups": 8,
         "act": "tanh", "dtype": "float32", "train": False},
        # a training step between two 256-wide layers
        {"name": "norm train 2^19x256 f32 tanh", "op": "norm", "n": 1 << 19, "s": 1, "channels": 256, "groups": 8,
         "act": "tanh", "dtype": "float32", "train": True},
        # a training step on fields over a 64 x 64 grid, channels last
        {"name": "norm train 8x4096x320 bf16 silu", "op": "norm", "n": 8, "s": 4096, "channels": 320, "groups": 32,
         "act": "silu", "dtype": "bfloat16", "train": True},
        # fields over ragged sets of points, rows that no vector load divides
        {"name": "norm train 5x1999x90 f16 identity", "op": "norm", "n": 5, "s": 1999, "channels": 90, "groups": 6,
         "act": "identity", "dtype": "float16", "train": True},
        # a physics-informed training step on 64-wide layers: value, two first and one second derivative a channel
        {"name": "jet norm train 2^19x64x4 tanh", "op": "jet", "n": 1 << 19, "channels": 64, "groups": 8, "n_dir": 2,
         "n_second": 1, "act": "tanh", "train": True},
        # the same for a basket of five assets, an odd number of points
        {"name": "jet norm train 30011x128x12 silu", "op": "jet", "n": 30011, "channels": 128, "groups": 4, "n_dir": 6,
         "n_second": 5, "act": "silu", "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("orthogonalize", "orthogonalize", "muon", "norm", "norm", "jet"))
    if op == "orthogonalize":
        dtype = rng.choice(("float32", "float32", "bfloat16", "float16"))
        rows, cols = _log_int(rng, 1, 4096), _log_int(rng, 1, 8192)
        batch = rng.randint(1, 5)
        while batch > 1 and _ns_flops(rows, cols) * batch > _ns_flops(1000, 771) * 4:
            batch -= 1
        while _ns_flops(rows, cols) > _ns_flops(2048, 8192):
            rows = rows * 3 // 4
        return {"op": op, "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}
    if op == "muon":
        return {"op": op, "width": _log_int(rng, 2, 256), "hidden": rng.randint(1, 3), "grid": rng.choice((3, 5, 8, 10, 20))}
    groups = rng.choice((1, 2, 4, 6, 8, 32))
    channels = groups * _log_int(rng, 8, max(8, 384 // groups))
    act, train = rng.choice(("tanh", "silu", "identity")), rng.random() < 0.7
    if op == "jet":
        n_dir, n_second = rng.choice(((2, 1), (2, 1), (6, 5)))
        n = _log_int(rng, 1, (1 << 27) // (channels * (1 + n_dir + n_second)))
        return {"op": op, "n": n, "channels": channels, "groups": groups, "n_dir": n_dir, "n_second": n_second,
                "act": act, "train": train}
    s = rng.choice((1, 1, _log_int(rng, 2, 16384)))
    n = _log_int(rng, 1, max(1, (1 << 26) // (channels * s)))
    return {"op": op, "n": n, "s": s, "channels": channels, "groups": groups, "act": act,
            "dtype": rng.choice(("float32", "bfloat16", "float16")), "train": train}


# ---- inputs -------------------------------------------------------------------------------------------------------

def _muon_shapes(case):
    """(rows, cols) of the parameters of a KAN [2, width, ..., width, 1] as its optimiser sees them: base weight,
    spline weight (one row an output) and spline scaler of each layer."""
    widths = [2] + [case["width"]] * case["hidden"] + [1]
    return [shape for i, o in zip(widths, widths[1:]) for shape in ((o, i), (o, i, case["grid"] + 3), (o, i))]


def _gradient(gen, shape, dtype=torch.float32):
    """A minibatch gradient: a part of low rank above noise of every direction."""
    *batch, m, n = shape
    rank = max(1, min(m, n) // 8)
    left = torch.randn(*batch, m, rank, device="cuda", generator=gen)
    right = torch.randn(*batch, rank, n, device="cuda", generator=gen)
    noise = torch.randn(*batch, m, n, device="cuda", generator=gen)
    return (1e-3 * (left @ right / rank ** 0.5 + 0.5 * noise)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)
    state = {"case": case}
    if case["op"] == "orthogonalize":
        lead = (case["batch"],) if case["batch"] > 1 else ()
        state["g"] = _gradient(gen, lead + (case["rows"], case["cols"]), DTYPES[case["dtype"]])
    elif case["op"] == "muon":
        shapes = _muon_shapes(case)
        flat = [(s[0], s[1] * (s[2] if len(s) == 3 else 1)) for s in shapes]
        state["params"] = [torch.nn.Parameter(0.1 * rand(*s)) for s in shapes]
        state["grads"] = [_gradient(gen, f).view(s) for f, s in zip(flat, shapes)]
        state["moments"] = [0.3 * _gradient(gen, f).view(s) for f, s in zip(flat, shapes)]
        if own:
            from pde_amd.optim import Muon
            opt = Muon(state["params"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, eps=NS_EPS)
            for p, g, m in zip(state["params"], state["grads"], state["moments"]):
                p.grad = g
                opt.state[p]["momentum_buffer"] = m
            state["opt"] = opt
    else:
        c = case["channels"]
        state["weight"] = torch.nn.Parameter(1 + 0.2 * rand(c))
        state["bias"] = torch.nn.Parameter(0.2 * rand(c))
        if case["op"] == "norm":
            lead = (case["n"],) if case["s"] == 1 else (case["n"], case["s"])
            dtype = DTYPES[case["dtype"]]
        else:
            lead, dtype = (case["n"],), torch.float32
        jets = (1 + case["n_dir"] + case["n_second"],) if case["op"] == "jet" else ()
        x = 0.7 * rand(*lead, c, *jets) + rand(c, *(1,) * len(jets))
        state["x"] = x.to(dtype).requires_grad_(case["train"])
        state["gy"] = (rand(*lead, c, *jets)).to(dtype) if case["train"] else None
    return state


# ---- plain forms --------------------------------------------------------------------------------------------------

def _ns_plain(g):
    """X <- a X + (b A + c A A) X with A = X X^T, five times, from X = G / (|G| + eps)."""
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.size(-2) > x.size(-1)
    x = x.transpose(-2, -1) if tall else x
    x = (x / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)).float()
    for _ in range(5):
        s = x @ x.transpose(-2, -1)
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.transpose(-2, -1) if tall else x).to(g.dtype)


def _muon_plain(p, g, m):
    """m <- mu m + (1 - mu) g; p <- (1 - lr decay) p - lr sqrt(max(1, rows / cols)) NS((1 - mu) g + mu m)."""
    m.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
    update = ((1 - MOMENTUM) * g + MOMENTUM * m).flatten(1)
    gain = max(1.0, update.size(0) / update.size(1)) ** 0.5
    p.data.mul_(1 - LR * DECAY).sub_(_ns_plain(update).view_as(p), alpha=LR * gain)
    return p, m


def _act_plain(u, act):
    """The activation and its first two derivatives."""
    if act == "identity":
        return u, torch.ones_like(u), torch.zeros_like(u)
    if act == "tanh":
        t = torch.tanh(u)
        d = 1 - t * t
        return t, d, -2 * t * d
    s = torch.sigmoid(u)
    d = s * (1 - s)
    return u * s, s + u * d, d * (2 + u * (1 - 2 * s))


def _norm_plain(x, gy, w, b, groups, act):
    n, c = x.size(0), x.size(-1)
    split = lambda v: v.float().reshape(n, -1, groups, c // groups)
    per = lambda v: v.view(groups, c // groups)
    mean = lambda v: v.mean((1, 3), keepdim=True)
    xs = split(x)
    xc = xs - mean(xs)
    r = torch.rsqrt(mean(xc * xc) + NORM_EPS)
    z = xc * r
    y, d, _ = _act_plain(z * per(w) + per(b), act)
    if gy is None:
        return y.reshape(x.shape).to(x.dtype)
    p = split(gy) * d
    q = p * per(w)
    gx = r * (q - mean(q) - z * mean(q * z))
    return {"y": y.reshape(x.shape).to(x.dtype), "gx": gx.reshape(x.shape).to(x.dtype),
            "gw": (p * z).sum((0, 1)).reshape(-1), "gb": p.sum((0, 1)).reshape(-1)}


def _jet_plain(x, w, b, groups, n_dir, n_second, act):
    """The norm by the chain rule, slot by slot: values, n_dir first derivatives, n_second second derivatives."""
    n, c, _ = x.shape
    v = x.reshape(n, groups, c // groups, -1)
    w, b = w.view(groups, -1, 1), b.view(groups, -1, 1)
    mean = lambda t: t.mean(2, keepdim=True)
    e = v - mean(v)
    xc, e1, e2 = e[..., :1], e[..., 1:1 + n_dir], e[..., 1 + n_dir:]
    r = torch.rsqrt(mean(xc * xc) + NORM_EPS)
    v1 = 2 * mean(xc * e1)
    r1 = -0.5 * r ** 3 * v1
    f1 = e1[..., :n_second]
    v2 = 2 * mean(f1 * f1 + xc * e2)
    r2 = -0.5 * r ** 3 * v2 + 0.75 * r ** 5 * v1[..., :n_second] ** 2
    u1 = w * (e1 * r + xc * r1)
    u2 = w * (e2 * r + 2 * f1 * r1[..., :n_second] + xc * r2)
    y, d, dd = _act_plain(w * xc * r + b, act)
    return torch.cat((y, d * u1, dd * u1[..., :n_second] ** 2 + d * u2), -1).reshape(x.shape)


def run(state):
    case = state["case"]
    if case["op"] == "orthogonalize":
        if own:
            from pde_amd import functional as K
            return K.orthogonalize(state["g"], eps=NS_EPS)
        return _ns_plain(state["g"])
    if case["op"] == "muon":
        if own:
            state["opt"].step()
            return state["params"], state["moments"]
        done = [_muon_plain(p, g, m) for p, g, m in zip(state["params"], state["grads"], state["moments"])]
        return [p for p, _ in done], [m for _, m in done]
    x, gy, w, b, groups, act = state["x"], state["gy"], state["weight"], state["bias"], case["groups"], case["act"]
    if own:
        from pde_amd import functional as K
        kind = {"identity": K.ACT_IDENTITY, "silu": K.ACT_SILU, "tanh": K.ACT_TANH}[act]
        with torch.set_grad_enabled(gy is not None):
            if case["op"] == "norm":
                y = K.group_norm_act(x, groups, w, b, NORM_EPS, kind)
            else:
                y = K.group_norm_act_jet(x, groups, w, b, NORM_EPS, kind, case["n_dir"], case["n_second"])
        if gy is None:
            return y
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    if case["op"] == "norm":
        with torch.no_grad():
            return _norm_plain(x, gy, w, b, groups, act)
    with torch.set_grad_enabled(gy is not None):
        y = _jet_plain(x, w, b, groups, case["n_dir"], case["n_second"], act)
    if gy is None:
        return y
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    return {"y": y, "gx": gx, "gw": gw, "gb": gb}


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def _ns_flops(rows, cols):
    """Multiply-adds of five steps, two operations each: half of X X^T, which is symmetric, once; every further product
    among symmetric matrices of the short side that commute (half of each): two powers a step, two more to carry the
    square on to the next step and one to compose the step with those before it; and the composed step times X."""
    m, n = min(rows, cols), max(rows, cols)
    return 2 * m * m * n * 1.5 + 2 * m ** 3 * 0.5 * (5 + 2 * 4 + 4)


def work(case):
    if case["op"] == "orthogonalize":
        k, size = case["batch"], DTYPES[case["dtype"]].itemsize
        return {"bytes": 2 * k * case["rows"] * case["cols"] * size, "flops": k * _ns_flops(case["rows"], case["cols"])}
    if case["op"] == "muon":
        flat = [(s[0], s[1] * (s[2] if len(s) == 3 else 1)) for s in _muon_shapes(case)]
        # weight and momentum read and written, gradient read
        return {"bytes": sum(5 * 4 * r * c for r, c in flat), "flops": sum(_ns_flops(r, c) for r, c in flat)}
    if case["op"] == "norm":
        values, size = case["n"] * case["s"] * case["channels"], DTYPES[case["dtype"]].itemsize
        flops = 30
    else:
        values, size = case["n"] * case["channels"] * (1 + case["n_dir"] + case["n_second"]), 4
        flops = 40
    # forward: x read, y written; a training step reads gy and writes gx as well
    return {"bytes": values * size * (4 if case["train"] else 2), "flops": values * flops * (3 if case["train"] else 1)}


# ---- in 64 bits, from the definitions -----------------------------------------------------------------------------

def _ns_exact(g):
    """phi(S) G with phi the composed polynomial of the squared singular values, built up in the Gram matrix alone."""
    a, b, c = COEFFICIENTS
    x = g.double()
    if x.size(-2) > x.size(-1):
        return _ns_exact(g.transpose(-2, -1)).transpose(-2, -1)
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + NS_EPS)
    s = x @ x.mT.contiguous()
    one = torch.eye(x.size(-2), dtype=torch.float64, device=x.device)
    phi = one
    for _ in range(5):
        q = a * one + s @ (b * one + c * s)
        phi, s = q @ phi, q @ s @ q
    return phi @ x


def _norm_exact(x, w, b, groups, act):
    """act(w (x - E x) / sqrt(V x + eps) + b) over the groups of a sample, by E x and E x^2 of x about its first value."""
    n, c = x.size(0), x.size(-1)
    v = x.reshape(n, -1, groups, c // groups).transpose(1, 2).reshape(n, groups, -1)
    v = v - v[..., :1].detach()
    m1 = v.sum(-1, keepdim=True) / v.size(-1)
    m2 = (v ** 2).sum(-1, keepdim=True) / v.size(-1)
    z = (v - m1) / (m2 - m1 ** 2 + NORM_EPS) ** 0.5
    z = z.reshape(n, groups, -1, c // groups).transpose(1, 2).reshape(x.shape)
    u = z * w + b
    return u if act == "identity" else u / (1 + torch.exp(-u)) if act == "silu" else 1 - 2 / (torch.exp(2 * u) + 1)


def _jet_exact(x, w, b, case):
    """Derivatives of the norm along the curve x + t x' + t^2 x'' / 2 at t = 0, by differentiating the values."""
    from torch.func import jvp
    f = lambda t: _norm_exact(t, w, b, case["groups"], case["act"])
    x0, n_dir = x[..., 0].clone(), case["n_dir"]
    slots, seconds = [f(x0)], []
    for d in range(n_dir):
        x1 = x[..., 1 + d]
        first = lambda t, t1: jvp(f, (t,), (t1,))[1]
        if d < case["n_second"]:
            y1, y2 = jvp(first, (x0, x1), (x1, x[..., 1 + n_dir + d]))
            seconds.append(y2)
        else:
            y1 = first(x0, x1)
        slots.append(y1)
    return torch.stack(slots + seconds, -1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orthogonalize":
        return _ns_exact(state["g"])
    if case["op"] == "muon":
        params, moments = [], []
        for p, g, m in zip(state["params"], state["grads"], state["moments"]):
            p, g, m = p.detach().double(), g.double(), m.double()
            m = m + (1 - MOMENTUM) * (g - m)
            nesterov = (g + MOMENTUM * (m - g)).flatten(1)
            r, c = nesterov.shape
            params.append(p - LR * (DECAY * p + max(1.0, r / c) ** 0.5 * _ns_exact(nesterov).view_as(p)))
            moments.append(m)
        return params, moments
    x, w, b = (state[k].detach().double() for k in ("x", "weight", "bias"))
    f = (lambda x, w, b: _norm_exact(x, w, b, case["groups"], case["act"])) if case["op"] == "norm" else \
        (lambda x, w, b: _jet_exact(x, w, b, case))
    if not case["train"]:
        return f(x, w, b)
    y, pull = torch.func.vjp(f, x, w, b)
    gx, gw, gb = pull(state["gy"].double())
    return {"y": y, "gx": gx, "gw": gw, "gb": gb}
