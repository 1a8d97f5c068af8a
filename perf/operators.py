"""Performance cases of the training operators: the optimizer step and the norms of a residual block.

Two kinds of call (``op``):

* ``adamw``  one AdamW step over many tensors at once (``gradient_norm`` where the gradients are
             clipped, then ``adamw_step``), with moments in float32 or in 8 bits;
* ``norm``   ``equivariant_norm``: the norm before the first block of a model;
* ``block``  ``gated_residual_norm``: the norm of a block's output, its gate, the residual sum and the
             norm before the next block.

The norms run forward (``order`` 0), with their gradients (1: training on energies) or with the
gradients of those gradients (2: training on forces, which are gradients themselves).

AdamW, for a gradient G scaled by the clipping coefficient c = min(1, max_norm / |G|) and the step t::

    m <- b1 m + (1 - b1) c G        v <- b2 v + (1 - b2) (c G)^2
    p <- (1 - lr wd) p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)

Eight-bit moments are kept in blocks of 256 values of the flat state (each tensor starts a block).
A block has the exponent byte f of its largest magnitude, raised by one where that lies above 1.75 in
its binade, and each value is a small floating number relative to 2^(f - 127): m with a sign, 4 exponent
and 3 mantissa bits (down to 2^-17), v with 5 exponent and 3 mantissa bits (down to 2^-33; a v above zero
is never stored as zero).  Values are rounded up or down at random, by 16 bits of a hash of the seed, the
step and the value's place, so that the small changes of a slow moving average are kept on average.

The norm of a row x with degrees l <= L, channels c and components m (mul_ir: per degree a [C, 2l+1]
block) is w_lc x_lcm rho, rho = (q + eps)^(-1/2), q the mean over degrees, channels and components (each
degree with the same weight).  The block's end is h = x + s sigmoid(gate_lc) norm(block; post), y =
norm(h; pre); x may have fewer degrees than the block (the missing ones are zero) or more (dropped).
"""
import itertools
import math
import os
import random
import sys

import torch

own = False

BLOCK = 256
LR, BETAS, EPS, DECAY = 2e-3, (0.9, 0.999), 1e-8, 1e-2
NORM_EPS = 1e-5
RESIDUAL_SCALE = 0.5
MASK = 0xFFFFFFFF


def listed():
    return [
        # a small model's optimizer step (40 tensors, 0.2 million parameters): launches and host work
        {"name": "adamw32_model_c64_l2", "op": "adamw", "bits": 32, "channels": 64, "lmax": 2, "species": 3,
         "max_norm": 0.0},
        # the benchmark's model (47 tensors, 1.5 million parameters), clipped as force training does
        {"name": "adamw32_clip_model_c128_l3", "op": "adamw", "bits": 32, "channels": 128, "lmax": 3, "species": 10,
         "max_norm": 10.0},
        # a large model: many matrices of millions of parameters, memory traffic only
        {"name": "adamw32_clip_large", "op": "adamw", "bits": 32, "tensors": 120, "elements": 1000000, "spread": 0.7,
         "max_norm": 1.0},
        # 8-bit moments: the benchmark's model
        {"name": "adamw8_model_c128_l3", "op": "adamw", "bits": 8, "channels": 128, "lmax": 3, "species": 10,
         "max_norm": 0.0},
        # hundreds of small tensors of odd sizes (biases, scales, per-element tables), clipped
        {"name": "adamw8_clip_ragged", "op": "adamw", "bits": 8, "tensors": 300, "elements": 2000, "spread": 2.0,
         "max_norm": 1.0},
        # a large model with 8-bit moments
        {"name": "adamw8_large", "op": "adamw", "bits": 8, "tensors": 120, "elements": 1000000, "spread": 0.7,
         "max_norm": 0.0},
        # the first norm of a small molecule's evaluation: launches and host work
        {"name": "norm_small_c64_l2", "op": "norm", "atoms": 50, "channels": 64, "lmax": 2, "order": 0},
        # the norm before a block with its gradients, a large structure
        {"name": "norm_grad_c128_l3", "op": "norm", "atoms": 16384, "channels": 128, "lmax": 3, "order": 1},
        # the end of a block, forward, of a large structure (relaxation, batched evaluation)
        {"name": "block_c128_l3", "op": "block", "atoms": 32768, "channels": 128, "lmax": 3, "input_lmax": 3,
         "gated": True, "next": True, "order": 0},
        # the first block of the benchmark's model (scalars in, every degree out), trained on energies
        {"name": "block_grad_c128_l0_l3", "op": "block", "atoms": 2048, "channels": 128, "lmax": 3, "input_lmax": 0,
         "gated": True, "next": True, "order": 1},
        # an odd number of channels and atoms, no norm behind it, trained on energies
        {"name": "block_grad_c70_l2", "op": "block", "atoms": 5003, "channels": 70, "lmax": 2, "input_lmax": 2,
         "gated": True, "next": False, "order": 1},
        # force training of the benchmark's model and a batch of structures: second derivatives
        {"name": "block_force_c128_l3", "op": "block", "atoms": 8192, "channels": 128, "lmax": 3, "input_lmax": 3,
         "gated": True, "next": True, "order": 2},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        tensors = _log_int(rng, 1, 400)
        return {"op": "adamw", "bits": rng.choice((32, 8)), "tensors": tensors,
                "elements": _log_int(rng, 1, min(2000000, 40000000 // tensors)), "spread": rng.choice((0.0, 0.7, 1.5)),
                "max_norm": rng.choice((0.0, 1.0, 10.0))}
    channels = rng.choice((_log_int(rng, 4, 300), 32, 64, 128, 256))
    lmax = rng.randint(0, 3)
    order = rng.randint(0, 2)
    atoms = _log_int(rng, 1, min(60000, 30000000 // (channels * (lmax + 1) ** 2 * (1 + order))))
    if rng.random() < 0.3:
        return {"op": "norm", "atoms": atoms, "channels": channels, "lmax": lmax, "order": order}
    return {"op": "block", "atoms": atoms, "channels": channels, "lmax": lmax, "input_lmax": rng.choice((0, lmax, 3)),
            "gated": rng.random() < 0.75, "next": rng.random() < 0.75, "order": order}


# ---------------------------------------------------------------------------------------------
# Sizes
# ---------------------------------------------------------------------------------------------

def _model_sizes(channels, lmax, species):
    """Element counts of the trained tensors of the two-interaction model with these settings."""
    columns = ((23, 4, 1), (51, 6, 1), (65, 7, 1), (65, 6, 1)) if lmax == 3 else ((11, 3, 1), (21, 4, 1), (23, 4, 1))
    counts = (4, 6, 7, 6) if lmax == 3 else (3, 4, 4)
    c, square = channels, channels * channels
    sizes = [c * species]
    for paths, in_counts, ups in ((lmax + 1, (1,) * (lmax + 1), 1), (sum(counts), counts, lmax + 1)):
        sizes += [square] * ups + [64 * 8, 64 * 64, 64 * 64, paths * c * 64]
        sizes += [square * k for k in in_counts] + [species * square]
    for degrees in (lmax + 1, 1):
        sizes += [species * k * c for group in columns[:degrees] for k in group] + [square] * degrees
    return sizes + [c, 16 * c, 16]


def _sizes(case):
    if "tensors" not in case:
        return _model_sizes(case["channels"], case["lmax"], case["species"])
    rng = random.Random(case["tensors"] * 1000003 + case["elements"])
    return [max(1, int(case["elements"] * math.exp(case["spread"] * max(-2.0, min(2.0, rng.gauss(0.0, 1.0))))))
            for _ in range(case["tensors"])]


def _widths(case):
    w = case["channels"] * (case["lmax"] + 1) ** 2
    return w, case["channels"] * (case.get("input_lmax", case["lmax"]) + 1) ** 2, case["channels"] * (case["lmax"] + 1)


def work(case):
    if case["op"] == "adamw":
        n = float(sum(_sizes(case)))
        # parameter read and written, gradient read; moments read and written (8 bits: also returned as
        # the values they stand for, two bytes each)
        return {"bytes": n * (12 + (16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4)), "flops": n * 16}
    n = float(case["atoms"])
    w, wx, wg = _widths(case)
    if case["op"] == "norm":
        rows = {0: 2 * w, 1: 4 * w, 2: 2 * w + 2 * w + 3 * w}[case["order"]]     # x, y | dy, dx | X, x", dy"
        return {"bytes": 4 * n * rows, "flops": n * w * (4, 12, 36)[case["order"]]}
    gate, nxt = (wg if case["gated"] else 0), (w if case["next"] else 0)
    rows = wx + w + gate + w + nxt                                   # x, block, gate; h, y
    if case["order"] >= 1:
        rows += w + nxt + wx + w + gate                              # dh, dy; dx, dblock, dgate
    if case["order"] == 2:
        rows += wx + w + gate + wx + w + gate + w + nxt              # cotangents; gradients to x, block, gate, dh, dy
    return {"bytes": 4 * n * rows, "flops": n * w * (12, 36, 110)[case["order"]]}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_adamw(case, seed, gen) if case["op"] == "adamw" else _prepare_norm(case, gen)


def _prepare_adamw(case, seed, gen):
    sizes = _sizes(case)
    padded = [-(-n // BLOCK) * BLOCK for n in sizes]
    starts = [0, *itertools.accumulate(padded)][:-1]
    total = sum(padded)
    # parameters and gradients of one flat buffer each, every tensor at a block's start
    param, grad = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    exp_avg, exp_avg_sq = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    rng = random.Random(seed)
    for n, at in zip(sizes, starts):
        level = 10.0 ** rng.uniform(-3.0, -1.0)          # each tensor's gradients have a scale of their own
        param[at:at + n].normal_(0.0, 0.1, generator=gen)
        spread = torch.randn(n, device="cuda", generator=gen).exp_()
        grad[at:at + n].normal_(0.0, level, generator=gen).mul_(spread)
        exp_avg[at:at + n].normal_(0.0, 0.3 * level, generator=gen).mul_(spread)
        exp_avg_sq[at:at + n] = spread.square_().mul_(level * level)
    step = rng.randint(1, 2000)
    progress = torch.zeros(len(sizes) + 1, 3, device="cuda", dtype=torch.float64)
    progress[:-1, 0], progress[:-1, 1], progress[:-1, 2] = step, BETAS[0] ** step, BETAS[1] ** step
    if case["bits"] == 8:
        zero = torch.zeros(1, device="cuda", dtype=torch.int64)
        exp_avg = _encode(exp_avg, zero, True)
        exp_avg_sq = _encode(exp_avg_sq, zero, False)
    return {"case": case, "sizes": sizes, "starts": starts, "param": param, "grad": grad,
            "params": [param[at:at + n] for n, at in zip(sizes, starts)],
            "grads": [grad[at:at + n] for n, at in zip(sizes, starts)],
            "exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq, "progress": progress, "seed": seed & 0x7FFFFFFF}


def _prepare_norm(case, gen):
    n, c, big = case["atoms"], case["channels"], case["lmax"]
    w, wx, wg = _widths(case)

    def rows(width, level=1.0):
        # atoms differ in scale with their number of neighbours
        return (torch.randn(n, width, device="cuda", generator=gen)
                * (level * torch.exp(0.4 * torch.randn(n, 1, device="cuda", generator=gen))))

    def weight():
        return 1.0 + 0.2 * torch.randn((big + 1) * c, device="cuda", generator=gen)

    s = {"case": case, "x": rows(wx), "dy": rows(w)}
    if case["op"] == "norm":
        s.update(post=None, pre=weight(), x2=rows(wx))
        leaves = ("x", "pre")
    else:
        s.update(block=rows(w, 2.0), gate=torch.randn(n, wg, device="cuda", generator=gen) if case["gated"] else None,
                 post=weight(), pre=weight() if case["next"] else None, dh=rows(w),
                 x2=rows(wx), block2=rows(w), gate2=rows(wg) if case["gated"] else None)
        leaves = ("x", "block", "gate", "post", "pre")
    if case["order"] >= 1:
        for k in leaves + (("dh", "dy") if case["order"] == 2 else ()):
            if s.get(k) is not None:
                s[k].requires_grad_()
    return s


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def run(s):
    return _run_adamw(s) if s["case"]["op"] == "adamw" else _run_norm(s)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ictc-o3-hp-ascend_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from ictc_o3 import operators
    return operators


def _run_adamw(s):
    case, clip, extra = s["case"], None, {}
    if own:
        ops = _package()
        if case["max_norm"]:
            clip = ops.gradient_norm(s["grads"], max_norm=case["max_norm"])
        ops.adamw_step(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], s["progress"], lr=LR, betas=BETAS,
                       eps=EPS, weight_decay=DECAY, clip=clip, seed=s["seed"])
        if case["bits"] == 8:
            exp_avg, exp_avg_sq = ops.moment_values(s["exp_avg"], s["exp_avg_sq"])
        else:
            exp_avg, exp_avg_sq = s["exp_avg"], s["exp_avg_sq"]
    else:
        if case["max_norm"]:
            clip = _plain_gradient_norm(s["grad"], case["max_norm"])
        exp_avg, exp_avg_sq = _plain_adamw(s, clip)
    if clip is not None:
        extra = {"clip": clip}
    return {"param": s["param"], "exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq, "progress": s["progress"], **extra}


def _run_norm(s):
    case = s["case"]
    if own:
        ops = _package()
        if case["op"] == "norm":
            h, y = None, ops.equivariant_norm(s["x"], s["pre"], channels=case["channels"], eps=NORM_EPS)
        else:
            h, y = ops.gated_residual_norm(s["x"], s["block"], s["gate"], s["post"], s["pre"],
                                           channels=case["channels"], residual_scale=RESIDUAL_SCALE, eps=NORM_EPS)
    else:
        h, y = _plain_block(s)
    return _with_gradients(s, h, y)


def _with_gradients(s, h, y):
    """The outputs with the gradients that the case's order asks for, by autograd."""
    case = s["case"]
    out = {"h": h, "y": y}
    if case["order"] == 0:
        return out
    tops = [(t, g) for t, g in ((h, s.get("dh")), (y, s["dy"])) if t is not None]
    heads, cots = [t for t, _ in tops], [g for _, g in tops]
    rows = [k for k in ("x", "block", "gate") if s.get(k) is not None]
    weights = [k for k in ("post", "pre") if s.get(k) is not None]
    if case["order"] == 1:
        names = rows + weights
        grads = torch.autograd.grad(heads, [s[k] for k in names], cots)
        return {**out, **{"d_" + k: g for k, g in zip(names, grads)}}
    # forces: gradients to the rows with a recorded graph; then the gradients of their product with
    # the force loss's cotangents
    first = torch.autograd.grad(heads, [s[k] for k in rows], cots, create_graph=True)
    out.update(("d_" + k, g.detach()) for k, g in zip(rows, first))
    # (a block without a norm behind it is linear in x: none of its first gradients depends on it)
    names = [k for k in rows if k != "x" or y is not None] + weights + \
        [k for k in ("dh", "dy") if any(s.get(k) is g for g in cots)]
    second = torch.autograd.grad(first, [s[k] for k in names], [s[k + "2"] for k in rows])
    out.update(("dd_" + k, g) for k, g in zip(names, second))
    return {k: None if v is None else v.detach() for k, v in out.items()}


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------

def _mix(x):
    """A 32-bit mixing of integers: shifts and odd multipliers, modulo 2^32."""
    x = x ^ (x >> 16)
    x = (x * 0xBB67AE85) & MASK
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & MASK
    return x ^ (x >> 16)


def _random_bits(total, seed, step):
    """32 bits for each place of the flat state, from the seed and the step."""
    key = _mix((seed + step * 0x9E3779B9) & MASK)
    place = torch.arange(total, device="cuda", dtype=torch.int64)
    return _mix((place + key) & MASK)


def _power(exponent):
    """2^exponent in float32 from whole numbers in [-126, 127]."""
    return ((exponent + 127) << 23).to(torch.int32).view(torch.float32)


def _encode(values, bits, signed):
    """(codes, block exponents) of a flat float32 state; bits: 16 random bits for each value."""
    size = values.abs().reshape(-1, BLOCK)
    top = ((size.amax(1).view(torch.int32) + 0x1FFFFF) >> 23).clamp(1, 253)
    x = size * _power(127 - top)[:, None]
    lowest = -14 if signed else -30
    exponent = ((x.view(torch.int32) >> 23) - 127).clamp(min=lowest)
    raised = (bits.to(torch.float32) * 2.0 ** -16).reshape(-1, BLOCK if bits.numel() > 1 else 1)
    code = (exponent - lowest) * 8 + torch.floor(x * _power(3 - exponent) + raised).to(torch.int32)
    values = values.reshape(-1, BLOCK)
    code = torch.where(values < 0, code + 128, code) if signed else torch.where(values > 0, code.clamp(min=1), code)
    return code.to(torch.uint8).reshape(-1), top.to(torch.uint8)


def _decode(coded, signed):
    codes, top = coded
    code = codes.to(torch.int32).reshape(-1, BLOCK)
    size = code & 127 if signed else code
    field = size >> 3
    x = ((size & 7) + torch.where(field > 0, 8, 0)).to(torch.float32)
    x = x * _power(field.clamp(min=1) - (18 if signed else 34))
    x = x * _power(top.to(torch.int32) - 127)[:, None]
    return (torch.where(code > 127, -x, x) if signed else x).reshape(-1)


def _plain_gradient_norm(grad, max_norm):
    norm = torch.sqrt((grad * grad).sum())
    return torch.stack((norm, (max_norm / norm).clamp(max=1.0)))


def _plain_adamw(s, clip):
    b1, b2 = BETAS
    small = s["case"]["bits"] == 8
    g = s["grad"] if clip is None else s["grad"] * clip[1]
    progress = s["progress"]
    progress[:-1] = torch.stack((progress[:-1, 0] + 1, progress[:-1, 1] * b1, progress[:-1, 2] * b2), 1)
    c1, c2 = (1 - progress[0, 1]).float(), (1 - progress[0, 2]).float()
    m = _decode(s["exp_avg"], True) if small else s["exp_avg"]
    v = _decode(s["exp_avg_sq"], False) if small else s["exp_avg_sq"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    s["param"].copy_(s["param"] * (1 - LR * DECAY) - LR * (m / c1) / (torch.sqrt(v / c2) + EPS))
    if not small:
        return s["exp_avg"].copy_(m), s["exp_avg_sq"].copy_(v)
    bits = _random_bits(m.numel(), s["seed"], progress[0, 0].to(torch.int64))
    m, v = _encode(m, bits & 0xFFFF, True), _encode(v, bits >> 16, False)
    s["exp_avg"][0].copy_(m[0])
    s["exp_avg"][1].copy_(m[1])
    s["exp_avg_sq"][0].copy_(v[0])
    s["exp_avg_sq"][1].copy_(v[1])
    return _decode(m, True).to(torch.bfloat16), _decode(v, False).to(torch.bfloat16)


def _degrees(x, channels, lmax):
    """The degree blocks [N, C, 2l+1] of rows in mul_ir order."""
    return [x[:, channels * l * l:channels * (l + 1) ** 2].reshape(-1, channels, 2 * l + 1) for l in range(lmax + 1)]


def _plain_norm(blocks, weight, channels):
    q = sum((b * b).mean((1, 2)) for b in blocks) / len(blocks)
    rho = 1.0 / torch.sqrt(q + NORM_EPS)
    return [b * rho[:, None, None] * w[None, :, None] for b, w in zip(blocks, weight.reshape(-1, channels))]


def _flat(blocks):
    return torch.cat([b.reshape(b.shape[0], -1) for b in blocks], 1)


def _plain_block(s):
    case = s["case"]
    c, lmax = case["channels"], case["lmax"]
    if case["op"] == "norm":
        return None, _flat(_plain_norm(_degrees(s["x"], c, lmax), s["pre"], c))
    post = _plain_norm(_degrees(s["block"], c, lmax), s["post"], c)
    if s["gate"] is not None:
        open_ = 1.0 / (1.0 + torch.exp(-s["gate"])).reshape(-1, lmax + 1, c)
        post = [b * open_[:, l, :, None] for l, b in enumerate(post)]
    w, wx, _ = _widths(case)
    x = s["x"][:, :w] if wx >= w else torch.cat((s["x"], s["x"].new_zeros(s["x"].shape[0], w - wx)), 1)
    h = x + RESIDUAL_SCALE * _flat(post)
    return h, (_flat(_plain_norm(_degrees(h, c, lmax), s["pre"], c)) if s["pre"] is not None else None)


# ---------------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_adamw(s) if case["op"] == "adamw" else _exact_norm(s)


def _exact_round(x, u, lowest):
    """Magnitudes of one state [blocks, 256] as the values their codes stand for; u in [0, 1)."""
    mantissa, top = torch.frexp(x.amax(1, keepdim=True))
    top = torch.where(mantissa > 0.875, top + 1, top) - 1            # the binade that holds the largest one
    _, e = torch.frexp(torch.where(x > 0, x, torch.ones_like(x)))
    unit = torch.exp2((torch.maximum(e - 1, top + lowest) - 3).double())
    return torch.floor(x / unit + u) * unit, unit


def _exact_values(coded, signed):
    code = coded[0].long().reshape(-1, BLOCK)
    size = code % 128 if signed else code
    field, lead = size // 8, (size >= 8).double()
    low = 14 if signed else 30
    x = (lead + (size % 8).double() / 8) * torch.exp2((field - (size >= 8).long()).double() - low)
    x = x * torch.exp2(coded[1].double() - 127)[:, None]
    return torch.where(code > 127, -x, x) if signed else x


def _exact_adamw(s):
    case, (b1, b2) = s["case"], BETAS
    g = s["grad"].double()
    out = {"clip": None}
    if case["max_norm"]:
        norm = g.square().sum().sqrt()
        scale = torch.clamp(case["max_norm"] / norm, max=1.0)
        out["clip"] = torch.stack((norm, scale))
        g = g * scale
    steps = s["progress"].clone()
    steps[:-1, 0] += 1
    steps[:-1, 1] *= b1
    steps[:-1, 2] *= b2
    t = int(steps[0, 0])
    small = case["bits"] == 8
    m = _exact_values(s["exp_avg"], True).reshape(-1) if small else s["exp_avg"].double()
    v = _exact_values(s["exp_avg_sq"], False).reshape(-1) if small else s["exp_avg_sq"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = s["param"].double()
    out["param"] = p - LR * DECAY * p - LR * m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + EPS)
    if small:
        bits = _random_bits(m.numel(), s["seed"], t).reshape(-1, BLOCK)
        m = m.reshape(-1, BLOCK)
        m = _exact_round(m.abs(), (bits % 65536).double() / 65536, -14)[0] * m.sign()
        before = v.reshape(-1, BLOCK)
        v, unit = _exact_round(before, (bits // 65536).double() / 65536, -30)
        v = torch.where((v == 0) & (before > 0), unit, v)
    out.update(exp_avg=m.reshape(-1), exp_avg_sq=v.reshape(-1), progress=steps)
    if out["clip"] is None:
        del out["clip"]
    return out


def _exact_norm(s):
    """The rows with one index per element (its degree, channel and weight), and autograd in 64 bits."""
    case = s["case"]
    c, lmax = case["channels"], case["lmax"]
    d = {k: v.detach().double().requires_grad_(v.requires_grad) if isinstance(v, torch.Tensor) else v
         for k, v in s.items()}
    l_of = torch.cat([torch.full((c * (2 * l + 1),), l, dtype=torch.int64) for l in range(lmax + 1)]).cuda()
    place = torch.cat([l * c + torch.arange(c).repeat_interleave(2 * l + 1) for l in range(lmax + 1)]).cuda()
    share = 1.0 / ((lmax + 1) * c * (2 * l_of + 1).double())

    def norm(v, weight):
        return v * weight[place] * (v.square() @ share + NORM_EPS).pow(-0.5).unsqueeze(1)

    if case["op"] == "norm":
        return _with_gradients(d, None, norm(d["x"], d["pre"]))
    u = norm(d["block"], d["post"])
    if d["gate"] is not None:
        u = u * torch.sigmoid(d["gate"])[:, place]
    both = min(d["x"].shape[1], u.shape[1])
    h = torch.nn.functional.pad(d["x"][:, :both], (0, u.shape[1] - both)) + RESIDUAL_SCALE * u
    return _with_gradients(d, h, norm(h, d["pre"]) if d["pre"] is not None else None)
