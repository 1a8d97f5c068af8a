"""Performance cases of the layers and the optimizer of a deep radial network.

Four kinds of call (``op``):

* ``layer_norm``   ``layer_norm`` over the last axis, with or without SiLU behind it: what stands between the
                   linear layers of a radial network (rows are edges), or before a readout (rows are atoms);
* ``embedding``    ``embedding``: a row of a table for each token (an atom's species, the pair of species of an
                   edge), times a scale, and the gradient of the table, summed over each row's tokens;
* ``orthogonal``   ``orthogonalize``: matrices' nearest (half-)orthogonal ones by Newton-Schulz products;
* ``muon``         ``muon_step``: one optimizer step over many matrices: moving average of the gradients, its
                   orthogonalisation, weight decay and update.

The norm of a row x of n values is y = f(w xh + b), xh = (x - mean) / sqrt(var + eps), var the mean of
(x - mean)^2, f the identity or SiLU.  It runs forward (``order`` 0), with its gradients (1: training on
energies) or with the gradients of those (2: training on forces, which are gradients themselves).

The embedding is y_i = s T[t_i], its gradient dT[v] = s sum over {i: t_i = v} of dy_i.

Newton-Schulz: X <- U / (|U|_F + eps), then five times X <- a X + (b A + c A^2) X with A = X X^T and
(a, b, c) = (3.4445, -4.7750, 2.0315); a matrix with more rows than columns is transposed around it.  The
optimizer's step of a parameter P with gradient G and moving average M::

    M <- beta M + (1 - beta) G          U = beta M + (1 - beta) G
    P <- (1 - lr wd) P - lr sqrt(max(1, rows / columns)) X(U)

The leading axes of a tensor with more than two count its matrices.
"""
import math
import os
import random
import sys

import torch

own = False

NORM_EPS = 1e-5
STEPS, EPS = 5, 1e-7
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
LR, BETA, DECAY = 0.02, 0.95, 0.01


def listed():
    return [
        # a hidden layer of the radial network of a small molecule's evaluation: launches and host work
        {"name": "ln_silu_small", "op": "layer_norm", "rows": 1250, "width": 64, "silu": True, "bias": True, "order": 0},
        # the benchmark graph's edges (2,048 atoms), trained on forces: second derivatives
        {"name": "ln_silu_force_w64", "op": "layer_norm", "rows": 105634, "width": 64, "silu": True, "bias": True,
         "order": 2},
        # scalar features of a large structure before a readout, trained on energies
        {"name": "ln_grad_w512", "op": "layer_norm", "rows": 32768, "width": 512, "silu": False, "bias": True,
         "order": 1},
        # an odd width without bias and with an activation
        {"name": "ln_silu_grad_w1001", "op": "layer_norm", "rows": 5003, "width": 1001, "silu": True, "bias": False,
         "order": 1},
        # the atoms' species of the benchmark's model: few rows, launches
        {"name": "embed_nodes_c128", "op": "embedding", "tokens": 2048, "rows": 10, "width": 128, "skew": 0.5,
         "order": 1},
        # the pairs of 10 species on the benchmark graph's edges: a thousand tokens to a row and more
        {"name": "embed_pairs_10", "op": "embedding", "tokens": 105634, "rows": 100, "width": 64, "skew": 1.0,
         "order": 1},
        # the pairs of 89 species on a large batch's edges: most rows rare, some with a tenth of the edges
        {"name": "embed_pairs_89", "op": "embedding", "tokens": 500001, "rows": 7921, "width": 64, "skew": 1.1,
         "order": 1},
        # a large table: wide rows, few tokens each
        {"name": "embed_large", "op": "embedding", "tokens": 65537, "rows": 50000, "width": 512, "skew": 0.7,
         "order": 1},
        # the matrices of a small model (C64, degrees to 2): many small problems
        {"name": "orthogonal_model_c64_l2", "op": "orthogonal", "channels": 64, "lmax": 2, "species": 3},
        # one step over the matrices of the benchmark's model (C128, degrees to 3, 10 species)
        {"name": "muon_model_c128_l3", "op": "muon", "channels": 128, "lmax": 3, "species": 10},
        # matrices of odd sizes, wide, tall, and a single row
        {"name": "orthogonal_ragged", "op": "orthogonal",
         "shapes": "1x77 5x5 17x300 63x65 100x41 129x127 130x130 7x3x40 200x333 511x257 1000x70 90x1501"},
        # a large model: for each of four layers six matrices of 1 and 4 million parameters
        {"name": "muon_large", "op": "muon", "repeat": 4,
         "shapes": "1024x1024 1024x1024 1024x1024 1024x1024 1024x4096 4096x1024"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("layer_norm", "embedding", "orthogonal", "muon"))
    if kind == "layer_norm":
        width = rng.choice((_log_int(rng, 1, 2000), 64, 128, 256, 512))
        order = rng.randint(0, 2)
        return {"op": kind, "rows": _log_int(rng, 1, 20000000 // (width * (1 + order))), "width": width,
                "silu": rng.random() < 0.5, "bias": rng.random() < 0.75, "order": order}
    if kind == "embedding":
        width = rng.choice((_log_int(rng, 1, 1000), 64, 128, 256))
        return {"op": kind, "tokens": _log_int(rng, 1, min(600000, 40000000 // width)),
                "rows": _log_int(rng, 1, min(60000, 30000000 // width)), "width": width,
                "skew": rng.choice((0.0, 0.5, 1.0, 1.3)), "order": rng.randint(0, 1)}
    shapes = []
    for _ in range(_log_int(rng, 1, 24)):
        rows, columns = _log_int(rng, 1, 700), _log_int(rng, 1, 700)
        lead = "%dx" % rng.randint(2, 12) if rows * columns < 20000 and rng.random() < 0.2 else ""
        shapes.append("%s%dx%d" % (lead, rows, columns))
    return {"op": kind, "shapes": " ".join(shapes)}


# ---------------------------------------------------------------------------------------------
# Sizes
# ---------------------------------------------------------------------------------------------

def _model_shapes(channels, lmax, species):
    """Shapes of the trained matrices of the two-interaction model with these settings."""
    c = channels
    counts = {2: (3, 4, 4), 3: (4, 6, 7, 6)}[lmax]
    shapes = []
    for paths, per_degree, ups in ((lmax + 1, (1,) * (lmax + 1), 1), (sum(counts), counts, lmax + 1)):
        shapes += [(c, c)] * ups + [(64, 8), (64, 64), (64, 64), (paths * c, 64)]
        shapes += [(c, k * c) for k in per_degree] + [(species, c, c)]
    return shapes + [(c, c)] * (lmax + 2) + [(16, c)]


def _shapes(case):
    if "shapes" not in case:
        return _model_shapes(case["channels"], case["lmax"], case["species"])
    return [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split()] * case.get("repeat", 1)


def work(case):
    if case["op"] == "layer_norm":
        n, w = float(case["rows"]), case["width"]
        # x, y | dy, dx | the cotangent of dx, the gradients to x and to dy
        values = n * w * (2, 4, 7)[case["order"]] + (w * (1 + case["bias"]) * (1, 2, 3)[case["order"]])
        return {"bytes": 4 * values, "flops": n * w * (8, 24, 60)[case["order"]]}
    if case["op"] == "embedding":
        n, w = float(case["tokens"]), case["width"]
        rows = n + min(n, case["rows"]) + ((n + case["rows"]) if case["order"] else 0)     # y, the table | dy, dT
        return {"bytes": 4 * rows * w + 8 * n, "flops": n * w * (1 + case["order"])}
    total, flops = 0.0, 0.0
    for s in _shapes(case):
        m, n, k = min(s[-2:]), max(s[-2:]), math.prod(s[:-2])
        total += k * m * n
        # the two symmetric products by half: A = X X^T and A^2; then (b A + c A^2) X
        flops += STEPS * k * (m * (m + 1.0) * n + m * (m + 1.0) * m + 2.0 * m * m * n)
    # U read, X written | P and M read and written, G read
    return {"bytes": 4 * total * (2 if case["op"] == "orthogonal" else 5), "flops": flops}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"layer_norm": _prepare_layer_norm, "embedding": _prepare_embedding, "orthogonal": _prepare_matrices,
            "muon": _prepare_matrices}[case["op"]](case, gen)


def _prepare_layer_norm(case, gen):
    n, w = case["rows"], case["width"]

    def rows():
        # edges differ in scale with their distance
        return (torch.randn(n, w, device="cuda", generator=gen)
                * torch.exp(0.4 * torch.randn(n, 1, device="cuda", generator=gen)))

    s = {"case": case, "x": rows() + 0.3, "dy": rows(), "x2": rows(),
         "weight": 1.0 + 0.2 * torch.randn(w, device="cuda", generator=gen),
         "bias": 0.2 * torch.randn(w, device="cuda", generator=gen) if case["bias"] else None}
    if case["order"] >= 1:
        for k in ("x", "weight", "bias") + (("dy",) if case["order"] == 2 else ()):
            if s[k] is not None:
                s[k].requires_grad_()
    return s


def _prepare_embedding(case, gen):
    n, v, w = case["tokens"], case["rows"], case["width"]
    share = torch.arange(1, v + 1, device="cuda", dtype=torch.float64).pow(-case["skew"])
    order = torch.randperm(v, device="cuda", generator=gen)
    places = torch.rand(n, device="cuda", dtype=torch.float64, generator=gen) * share.sum()
    tokens = order[torch.searchsorted(share.cumsum(0), places).clamp(max=v - 1)]
    table = torch.randn(v, w, device="cuda", generator=gen)
    return {"case": case, "tokens": tokens, "table": table.requires_grad_(case["order"] >= 1), "scale": math.sqrt(w),
            "dy": torch.randn(n, w, device="cuda", generator=gen)}


def _prepare_matrices(case, gen):
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    total = sum(sizes)
    s = {"case": case, "shapes": shapes}
    for name, scale in (("grad", 1e-3), ("momentum", 5e-4), ("param", 0.05)):
        s[name] = torch.randn(total, device="cuda", generator=gen).mul_(scale)
        s[name + "s"] = [t.view(shape) for t, shape in zip(s[name].split(sizes), shapes)]
    # gradients of a layer are products of few large and many small directions
    for g, m in zip(s["grads"], s["momentums"]):
        level = torch.exp(torch.randn(g.shape[-1], device="cuda", generator=gen))
        g.mul_(level)
        m.mul_(level)
    return s


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def run(s):
    return {"layer_norm": _run_layer_norm, "embedding": _run_embedding, "orthogonal": _run_orthogonal,
            "muon": _run_muon}[s["case"]["op"]](s)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ictc-o3-hp-ascend_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from ictc_o3 import operators
    return operators


def _run_layer_norm(s):
    if own:
        y = _package().layer_norm(s["x"], s["weight"], s["bias"], eps=NORM_EPS,
                                  activation="silu" if s["case"]["silu"] else None)
        return _with_gradients(s, y)
    return _plain_layer_norm(s)


def _with_gradients(s, y):
    """The outputs with the gradients that the case's order asks for, by autograd."""
    if s["case"]["order"] == 0:
        return {"y": y}
    weights = [k for k in ("weight", "bias") if s[k] is not None]
    if s["case"]["order"] == 1:
        names = ["x"] + weights
        grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
        return {"y": y.detach(), **{"d_" + k: g for k, g in zip(names, grads)}}
    # forces: the gradient to the rows with a recorded graph; then the gradients of its product with
    # the force loss's cotangent (without an activation the bias does not take part in them)
    first, = torch.autograd.grad(y, s["x"], s["dy"], create_graph=True)
    names = ["x", "weight"] + (["bias"] if s["bias"] is not None and s["case"]["silu"] else []) + ["dy"]
    second = torch.autograd.grad(first, [s[k] for k in names], s["x2"])
    return {"y": y.detach(), "d_x": first.detach(), **{"dd_" + k: g for k, g in zip(names, second)}}


def _run_embedding(s):
    if own:
        y = _package().embedding(s["tokens"], s["table"], scale=s["scale"])
        if s["case"]["order"] == 0:
            return {"y": y}
        return {"y": y.detach(), "d_table": torch.autograd.grad(y, s["table"], s["dy"])[0]}
    out = {"y": s["table"].detach()[s["tokens"]] * s["scale"]}
    if s["case"]["order"]:
        summed = torch.zeros_like(s["table"], requires_grad=False).index_add_(0, s["tokens"], s["dy"])
        out["d_table"] = summed * s["scale"]
    return out


def _run_orthogonal(s):
    if own:
        return _package().orthogonalize(s["grads"], steps=STEPS, eps=EPS)
    return _plain_orthogonal(s["grads"])


def _run_muon(s):
    if own:
        _package().muon_step(s["params"], s["grads"], s["momentums"], lr=LR, beta=BETA, nesterov=True,
                             weight_decay=DECAY, steps=STEPS, eps=EPS)
        return {"param": s["param"], "momentum": s["momentum"]}
    s["momentum"].copy_(BETA * s["momentum"] + (1 - BETA) * s["grad"])
    flat = BETA * s["momentum"] + (1 - BETA) * s["grad"]
    sizes = [g.numel() for g in s["grads"]]
    update = _plain_orthogonal([u.view(shape) for u, shape in zip(flat.split(sizes), s["shapes"])])
    scaled = [x.reshape(-1) * math.sqrt(max(1.0, x.shape[-2] / x.shape[-1])) for x in update]
    s["param"].copy_((1 - LR * DECAY) * s["param"] - LR * torch.cat(scaled))
    return {"param": s["param"], "momentum": s["momentum"]}


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------

def _plain_layer_norm(s):
    """The formulas of the norm, of its gradients and of theirs, J the symmetric Jacobian of xh by x."""
    case, w = s["case"], s["weight"].detach()
    x, dy, u = s["x"].detach(), s["dy"].detach(), s["x2"]

    def mean(v):
        return v.mean(1, keepdim=True)

    xc = x - mean(x)
    rho = 1.0 / torch.sqrt(mean(xc * xc) + NORM_EPS)
    xh = xc * rho
    z = xh * w if s["bias"] is None else xh * w + s["bias"].detach()
    if case["silu"]:
        open_ = 1.0 / (1.0 + torch.exp(-z))
        y = z * open_
    else:
        open_, y = None, z
    if case["order"] == 0:
        return {"y": y}

    def jacobian(v):
        return rho * (v - mean(v) - xh * mean(v * xh))

    slope = 1.0 if open_ is None else open_ * (1.0 + z * (1.0 - open_))
    dz = dy * slope
    out = {"y": y, "d_x": jacobian(w * dz)}
    if case["order"] == 1:
        out["d_weight"] = (dz * xh).sum(0)
        if s["bias"] is not None:
            out["d_bias"] = dz.sum(0)
        return out
    t, e = jacobian(u), w * dz
    a, c = u - mean(u), e - mean(e)
    along, across = mean(xh * a), mean(xh * c)
    dd_x = -rho * rho * (xh * (mean(a * c) - 3.0 * along * across) + across * a + along * c)
    dd_w = t * dz
    if open_ is not None:
        bend = w * t * dy * (open_ * (1.0 - open_) * (2.0 + z * (1.0 - 2.0 * open_)))
        dd_x = dd_x + jacobian(w * bend)
        dd_w = dd_w + bend * xh
        if s["bias"] is not None:
            out["dd_bias"] = bend.sum(0)
    return {**out, "dd_x": dd_x, "dd_weight": dd_w.sum(0), "dd_dy": w * t * slope}


def _plain_orthogonal(matrices):
    """Newton-Schulz of matrices of any shapes, those of one shape stacked."""
    flat = [m.reshape(-1, m.shape[-2], m.shape[-1]) for m in matrices]
    flat = [m.transpose(1, 2) if m.shape[1] > m.shape[2] else m for m in flat]
    places = {}
    [places.setdefault(m.shape[1:], []).append(i) for i, m in enumerate(flat)]
    results = [None] * len(flat)
    for at in places.values():
        done = _plain_newton_schulz(torch.cat([flat[i] for i in at]))
        for i, x in zip(at, done.split([flat[i].shape[0] for i in at])):
            x = x.transpose(1, 2) if matrices[i].shape[-2] > matrices[i].shape[-1] else x
            results[i] = x.reshape(matrices[i].shape)
    return results


def _plain_newton_schulz(x):
    a, b, c = COEFFICIENTS
    norm = torch.sqrt((x.double() * x.double()).sum((1, 2), keepdim=True))     # (sums of a million squares)
    x = x * (1.0 / (norm + EPS)).float()
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x


# ---------------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        d = {k: v.detach().double().requires_grad_(v.requires_grad) if isinstance(v, torch.Tensor) else v
             for k, v in s.items()}
        var, middle = torch.var_mean(d["x"], 1, correction=0, keepdim=True)
        z = d["weight"] * ((d["x"] - middle) / (var + NORM_EPS).sqrt())
        z = z if d["bias"] is None else z + d["bias"]
        return _with_gradients(d, z * torch.sigmoid(z) if case["silu"] else z)
    if case["op"] == "embedding":
        out = {"y": s["table"].detach().double().index_select(0, s["tokens"]).mul_(s["scale"])}
        if case["order"]:
            # tokens in order of their rows; a row's sum is a difference of running sums
            order = torch.argsort(s["tokens"], stable=True)
            ends = torch.bincount(s["tokens"], minlength=case["rows"]).cumsum(0)
            columns = [torch.nn.functional.pad(part[order].double().cumsum(0), (0, 0, 1, 0))
                       for part in s["dy"].split(64, 1)]
            starts = torch.nn.functional.pad(ends[:-1], (1, 0))
            out["d_table"] = torch.cat([part[ends] - part[starts] for part in columns], 1) * s["scale"]
        return out
    if case["op"] == "orthogonal":
        return [_exact_orthogonal(g) for g in s["grads"]]
    params, momenta = [], []
    for p, g, m in zip(s["params"], s["grads"], s["momentums"]):
        m = m.double().lerp(g.double(), 1 - BETA)
        x = _exact_orthogonal(g.double().lerp(m, BETA))
        rate = LR * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5
        params.append((p.double() * (1 - LR * DECAY) - rate * x).reshape(-1))
        momenta.append(m.reshape(-1))
    return {"param": torch.cat(params), "momentum": torch.cat(momenta)}


def _exact_orthogonal(u):
    """One matrix at a time, the polynomial in Horner's form on the shorter side."""
    a, b, c = COEFFICIENTS
    results = []
    for x in u.double().reshape(-1, *u.shape[-2:]):
        x = x / (torch.linalg.matrix_norm(x) + EPS)
        side = x.shape[0] <= x.shape[1]
        one = torch.eye(min(x.shape), device=x.device, dtype=x.dtype)
        for _ in range(STEPS):
            gram = x @ x.mT if side else x.mT @ x
            inner = a * one + gram @ (b * one + c * gram)
            x = inner @ x if side else x @ inner
        results.append(x)
    return torch.stack(results).reshape(u.shape)
