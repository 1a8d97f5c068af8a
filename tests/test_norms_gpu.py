"""The norms of a residual block against plain float64 formulas on the CPU: values, gradients, the
gradients of gradients (force training's), a third derivative, and the same gradients against central
differences of the float64 values.

Tolerances are the suite's 1e-5 of the largest entry: a statistic is a sum of at most 16 terms a thread and
ten levels of pairwise sums behind that (30 u, u = 6e-8, of the sum of magnitudes), its inverse root halves
that, and a second derivative multiplies three of them; weight gradients add rows in groups of at most a
few dozen before 64-bit sums.
"""
import pytest
import torch

from conftest import assert_rel

pytestmark = pytest.mark.gpu

EPS = 1e-5
# channels (a part of a wave, a whole one, two waves with six or all of the second's lanes, more than four), lmax, rows
SHAPES = [(1, 0, 1), (3, 1, 5), (16, 2, 33), (48, 3, 20), (64, 3, 7), (40, 1, 9), (70, 2, 130), (128, 3, 65),
          (129, 1, 17), (300, 3, 9), (1024, 0, 3), (5, 3, 3000)]


def _degrees(x, c, lmax):
    return [x[:, c * l * l:c * (l + 1) ** 2].reshape(-1, c, 2 * l + 1) for l in range(lmax + 1)]


def _norm(x, w, c, lmax):
    blocks = _degrees(x, c, lmax)
    q = sum(b.square().mean(dim=(1, 2)) for b in blocks) / len(blocks)
    return torch.cat([(b * w.reshape(-1, c)[l][None, :, None] / (q + EPS).sqrt()[:, None, None]).reshape(len(x), -1)
                      for l, b in enumerate(blocks)], 1)


def _block_end(x, block, gate, post, pre, c, lmax, scale):
    n = _norm(block, post, c, lmax)
    if gate is not None:
        n = torch.cat([(b * torch.sigmoid(gate).reshape(-1, lmax + 1, c)[:, l, :, None]).reshape(len(x), -1)
                       for l, b in enumerate(_degrees(n, c, lmax))], 1)
    width = n.shape[1]
    x = x[:, :width] if x.shape[1] >= width else torch.nn.functional.pad(x, (0, width - x.shape[1]))
    h = x + scale * n
    return h, None if pre is None else _norm(h, pre, c, lmax)


def _inputs(c, lmax, rows, seed, input_lmax=None, gated=True, behind=True):
    g = torch.Generator().manual_seed(seed)
    width, places = c * (lmax + 1) ** 2, c * (lmax + 1)
    wide = width if input_lmax is None else c * (input_lmax + 1) ** 2
    draw = lambda *s: torch.randn(*s, generator=g) * torch.exp(0.3 * torch.randn(s[0], 1, generator=g))   # noqa: E731
    return {"x": draw(rows, wide), "block": 2 * draw(rows, width),
            "gate": torch.randn(rows, places, generator=g) if gated else None,
            "post": 1 + 0.2 * torch.randn(places, generator=g),
            "pre": 1 + 0.2 * torch.randn(places, generator=g) if behind else None,
            "dh": draw(rows, width), "dy": draw(rows, width), "cx": draw(rows, wide), "cb": draw(rows, width),
            "cg": draw(rows, places)}


def _leaves(d, device, dtype):
    return {k: None if v is None else v.to(device=device, dtype=dtype).requires_grad_() for k, v in d.items()}


def _all_orders(t, h, y):
    """Values, first gradients and second gradients of one evaluation."""
    heads = [(o, t[k]) for o, k in ((h, "dh"), (y, "dy")) if o is not None]
    names = [k for k in ("x", "block", "gate", "post", "pre") if t[k] is not None]
    first = torch.autograd.grad([o for o, _ in heads], [t[k] for k in names], [c for _, c in heads], retain_graph=True)
    out = {"h": h, "y": y, **{"d" + k: g for k, g in zip(names, first)}}
    rows = [k for k in names if k in ("x", "block", "gate")]
    again = torch.autograd.grad([o for o, _ in heads], [t[k] for k in rows], [c for _, c in heads], create_graph=True)
    pairs = [(g, t[{"x": "cx", "block": "cb", "gate": "cg"}[k]].detach()) for k, g in zip(rows, again)]
    names += [k for o, k in ((h, "dh"), (y, "dy")) if o is not None]
    second = torch.autograd.grad([g for g, _ in pairs], [t[k] for k in names], [c for _, c in pairs], allow_unused=True)
    out.update({"dd" + k: g for k, g in zip(names, second)})
    return out


def _compare(got, want):
    assert got.keys() == want.keys()
    for k, w in want.items():
        if w is None:
            assert got[k] is None or not got[k].any(), k
            continue
        g = got[k]
        if g is None:
            assert not w.any(), k
            continue
        assert_rel(g, w, what=k)


@pytest.mark.parametrize("c,lmax,rows", SHAPES)
def test_norm_every_order(gpu, c, lmax, rows):
    from ictc_o3 import equivariant_norm
    d = _inputs(c, lmax, rows, c + rows)
    d = {"x": d["x"], "block": None, "gate": None, "post": None, "pre": d["pre"], "dy": d["dy"], "cx": d["cx"]}
    t, ref = _leaves(d, gpu, torch.float32), _leaves(d, "cpu", torch.float64)
    _compare(_all_orders(t, None, equivariant_norm(t["x"], t["pre"], channels=c, eps=EPS)),
             _all_orders(ref, None, _norm(ref["x"], ref["pre"], c, lmax)))


@pytest.mark.parametrize("gated,behind", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("c,lmax,rows", SHAPES)
def test_block_end_every_order(gpu, c, lmax, rows, gated, behind):
    from ictc_o3 import gated_residual_norm
    d = _inputs(c, lmax, rows, 10 * c + rows, gated=gated, behind=behind)
    t, ref = _leaves(d, gpu, torch.float32), _leaves(d, "cpu", torch.float64)
    got = gated_residual_norm(t["x"], t["block"], t["gate"], t["post"], t["pre"], channels=c, residual_scale=0.7, eps=EPS)
    want = _block_end(*[ref[k] for k in ("x", "block", "gate", "post", "pre")], c, lmax, 0.7)
    _compare(_all_orders(t, *got), _all_orders(ref, *want))


@pytest.mark.parametrize("lmax,input_lmax", [(3, 0), (2, 1), (0, 3), (1, 2), (0, 5)])
def test_features_of_other_degrees(gpu, lmax, input_lmax):
    """Missing degrees are zero, further ones are left out (and their gradient is zero)."""
    from ictc_o3 import gated_residual_norm
    c, rows = 70, 41
    for behind in (True, False):
        d = _inputs(c, lmax, rows, 3, input_lmax=input_lmax, behind=behind)
        t, ref = _leaves(d, gpu, torch.float32), _leaves(d, "cpu", torch.float64)
        got = gated_residual_norm(t["x"], t["block"], t["gate"], t["post"], t["pre"], channels=c, eps=EPS)
        want = _block_end(*[ref[k] for k in ("x", "block", "gate", "post", "pre")], c, lmax, 1.0)
        _compare(_all_orders(t, *got), _all_orders(ref, *want))


def test_only_one_result_is_used(gpu):
    """Gradients through h alone and through y alone."""
    from ictc_o3 import gated_residual_norm
    c, lmax, rows = 20, 2, 50
    d = _inputs(c, lmax, rows, 5)
    for use in (0, 1):
        t, ref = _leaves(d, gpu, torch.float32), _leaves(d, "cpu", torch.float64)
        for k in ("dh", "dy"):
            t[k], ref[k] = t[k].detach(), ref[k].detach()
        grads = []
        for s, out in ((t, gated_residual_norm(*[t[k] for k in ("x", "block", "gate", "post", "pre")], channels=c,
                                               eps=EPS)),
                       (ref, _block_end(*[ref[k] for k in ("x", "block", "gate", "post", "pre")], c, lmax, 1.0))):
            names = ["x", "block", "gate", "post"] + ["pre"] * use
            first = torch.autograd.grad(out[use], [s[k] for k in names], s["dy"], create_graph=True)
            second = torch.autograd.grad(first[1], [s["block"], s["gate"], s["post"]], s["cb"].detach())
            grads.append(dict(enumerate([*first, *second])))
        _compare(*grads)


def test_gradients_against_differences(gpu):
    from ictc_o3 import gated_residual_norm
    c, lmax, rows, step = 33, 3, 40, 1e-5
    d = _inputs(c, lmax, rows, 8)
    t = _leaves(d, gpu, torch.float32)
    names = ("x", "block", "gate", "post", "pre")
    h, y = gated_residual_norm(*[t[k] for k in names], channels=c, eps=EPS)
    grads = torch.autograd.grad([h, y], [t[k] for k in names], [t["dh"], t["dy"]])
    ref = {k: v.double() for k, v in d.items()}
    gen = torch.Generator().manual_seed(1)
    for k, g in zip(names, grads):
        along = torch.randn(ref[k].shape, generator=gen, dtype=torch.float64)
        value = []
        for sign in (1, -1):
            at = {**ref, k: ref[k] + sign * step * along}
            a, b = _block_end(*[at[n] for n in names], c, lmax, 1.0)
            value.append(float((a * ref["dh"]).sum() + (b * ref["dy"]).sum()))
        got = g.double().cpu()
        # the difference's own error: step^2 of the third derivative, and 64-bit rounding of the sums over the step
        assert abs(float((got * along).sum()) - (value[0] - value[1]) / (2 * step)) <= 1e-5 * float(
            (got * along).abs().sum())


def test_third_derivative_and_weight_cotangents(gpu):
    """A derivative of the second gradients, and cotangents of weight gradients (composed formulas)."""
    from ictc_o3 import gated_residual_norm
    c, lmax, rows = 6, 2, 11
    d = _inputs(c, lmax, rows, 9)
    out = []
    for device, dtype in ((gpu, torch.float32), ("cpu", torch.float64)):
        t = _leaves(d, device, dtype)
        names = ("x", "block", "gate", "post", "pre")
        if dtype == torch.float32:
            h, y = gated_residual_norm(*[t[k] for k in names], channels=c, eps=EPS)
        else:
            h, y = _block_end(*[t[k] for k in names], c, lmax, 1.0)
        first = torch.autograd.grad([h, y], [t[k] for k in names], [t["dh"], t["dy"]], create_graph=True)
        second = torch.autograd.grad([first[1], first[3], first[4]], [t["x"], t["block"], t["gate"]],
                                     [t["cb"].detach(), torch.ones_like(first[3]), torch.ones_like(first[4])],
                                     create_graph=True)
        third = torch.autograd.grad([s.square().sum() for s in second], [t[k] for k in names])
        out.append(dict(enumerate([*second, *third])))
    _compare(*out)


def test_rotations_commute(gpu):
    """An orthogonal mixing of each degree's components, before or after."""
    from ictc_o3 import gated_residual_norm
    c, lmax, rows = 24, 3, 20
    d = {k: v.to(gpu) for k, v in _inputs(c, lmax, rows, 12).items()}
    gen = torch.Generator().manual_seed(2)
    q = [torch.linalg.qr(torch.randn(2 * l + 1, 2 * l + 1, generator=gen, dtype=torch.float64))[0].float().to(gpu)
         for l in range(lmax + 1)]
    turn = lambda v: torch.cat([(b @ q[l]).reshape(rows, -1) for l, b in enumerate(_degrees(v, c, lmax))], 1)   # noqa: E731
    weights = [d["gate"], d["post"], d["pre"]]
    h, y = gated_residual_norm(d["x"], d["block"], *weights, channels=c, eps=EPS)
    h2, y2 = gated_residual_norm(turn(d["x"]), turn(d["block"]), *weights, channels=c, eps=EPS)
    assert_rel(h2, turn(h), what="h")
    assert_rel(y2, turn(y), what="y")


def test_empty_rows(gpu):
    """Rows of zeros (atoms without neighbours) and no rows at all."""
    from ictc_o3 import equivariant_norm, gated_residual_norm
    c, lmax = 16, 2
    d = _inputs(c, lmax, 9, 4)
    d["block"][3] = 0.0
    d["block"][5], d["x"][5] = 0.0, 0.0
    t, ref = _leaves(d, gpu, torch.float32), _leaves(d, "cpu", torch.float64)
    names = ("x", "block", "gate", "post", "pre")
    got = _all_orders(t, *gated_residual_norm(*[t[k] for k in names], channels=c, eps=EPS))
    want = _all_orders(ref, *_block_end(*[ref[k] for k in names], c, lmax, 1.0))
    for k, w in want.items():
        for row in range(9) if w.dim() == 2 else [...]:
            assert_rel(got[k][row], w[row], what=f"{k} row {row}")
    none = {k: v[:0] if v.dim() == 2 else v for k, v in d.items()}
    t = _leaves(none, gpu, torch.float32)
    h, y = gated_residual_norm(*[t[k] for k in names], channels=c, eps=EPS)
    assert h.shape == y.shape == t["block"].shape
    grads = torch.autograd.grad([h, y], [t[k] for k in names], [t["dh"], t["dy"]])
    assert not grads[3].any() and not grads[4].any()
    assert equivariant_norm(t["x"], t["pre"], channels=c).shape == t["x"].shape


def test_values_that_are_not_finite_stay_in_their_row(gpu):
    from ictc_o3 import gated_residual_norm
    d = {k: v.to(gpu) for k, v in _inputs(70, 1, 12, 6).items()}
    names = ("x", "block", "gate", "post", "pre")
    h, y = gated_residual_norm(*[d[k] for k in names], channels=70)
    d["block"][4, 7] = float("nan")
    d["x"][9, 3] = float("inf")
    h2, y2 = gated_residual_norm(*[d[k] for k in names], channels=70)
    keep = [i for i in range(12) if i not in (4, 9)]
    assert torch.equal(h[keep], h2[keep]) and torch.equal(y[keep], y2[keep])
    assert h2[4].isnan().all() and not torch.isfinite(h2[9, 3])


def test_weight_gradients_repeat_bit_for_bit(gpu):
    from ictc_o3 import gated_residual_norm
    d = _inputs(128, 3, 3000, 7)
    t = _leaves(d, gpu, torch.float32)
    names = ("x", "block", "gate", "post", "pre")
    runs = []
    for _ in range(3):
        h, y = gated_residual_norm(*[t[k] for k in names], channels=128)
        runs.append(torch.autograd.grad([h, y], [t[k] for k in names], [t["dh"], t["dy"]]))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_strided_operands_and_streams(gpu):
    from ictc_o3 import equivariant_norm
    c, lmax, rows = 16, 1, 30
    wide = torch.randn(rows, 2 * c * 4, device=gpu)
    w = torch.randn(2, c, device=gpu)
    want = _norm(wide[:, ::2].double().cpu(), w.double().cpu(), c, lmax)
    assert_rel(equivariant_norm(wide[:, ::2], w, channels=c, eps=EPS), want)
    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        out = equivariant_norm(wide[:, ::2], w, channels=c, eps=EPS)
    torch.cuda.current_stream(gpu).wait_stream(side)
    assert_rel(out, want)


def test_refusals(gpu):
    from ictc_o3 import equivariant_norm, gated_residual_norm
    x, w = torch.zeros(4, 16 * 4, device=gpu), torch.ones(32, device=gpu)
    gate = torch.zeros(4, 32, device=gpu)
    gated_residual_norm(x, x, gate, w, w, channels=16)
    for call in (lambda: equivariant_norm(x, w[:16], channels=16), lambda: equivariant_norm(x, w, channels=15),
                 lambda: equivariant_norm(x, w, channels=0), lambda: equivariant_norm(x, w, channels=16, eps=0.0),
                 lambda: equivariant_norm(x.double(), w.double(), channels=16),
                 lambda: equivariant_norm(x.cpu(), w.cpu(), channels=16),
                 lambda: equivariant_norm(x[0], w, channels=16),
                 lambda: equivariant_norm(torch.zeros(2, 25, device=gpu), torch.ones(5, device=gpu), channels=1),
                 lambda: equivariant_norm(torch.zeros(2, 1025, device=gpu), torch.ones(1025, device=gpu), channels=1025),
                 lambda: gated_residual_norm(x[:3], x, gate, w, w, channels=16),
                 lambda: gated_residual_norm(x, x, gate[:, :16], w, w, channels=16),
                 lambda: gated_residual_norm(x, x, None, w[:16], w, channels=16),
                 lambda: gated_residual_norm(x, x, None, w, w.reshape(4, 8), channels=16),
                 lambda: gated_residual_norm(x, x, None, w, w, channels=16, residual_scale=float("nan"))):
        with pytest.raises(ValueError):
            call()
