"""Layer norm against plain float64 formulas on the CPU: values, gradients, the gradients of gradients (force
training's), a third derivative, rows with a large mean or one large entry, empty inputs, strides, another
stream, captured passes and refusals.

Tolerances are the suite's 1e-5 of the largest entry.  Sums, means and projections are in 64 bits; per element
about ten float32 operations remain (u = 6e-8 each, an exponential's 2 u times its slope), products of at most
four of them in a second derivative, and weight gradients add rows in float32 in groups of at most a few
hundred before 64-bit sums: under 2e-6.
"""
import pytest
import torch

from conftest import assert_rel

pytestmark = pytest.mark.gpu

EPS = 1e-5
# width (one column, parts of a group of four, parts of a wave, whole ones, two and four groups a thread, rows of
# 4 and 16 waves), rows (one, less than a workgroup's, more than the workgroups with partial sums hold)
SHAPES = [(1, 3), (2, 9), (3, 300), (4, 1), (5, 70), (7, 2000), (16, 33), (63, 17), (64, 20000), (65, 40), (128, 130),
          (255, 9), (256, 65), (257, 33), (510, 12), (512, 40), (513, 20), (601, 37), (768, 5000), (769, 6), (1001,
          21), (1024, 9), (1025, 5), (2048, 6), (2050, 7), (4096, 3), (4099, 5), (8192, 2)]


def _formula(x, w, b, silu):
    xc = x - x.mean(-1, keepdim=True)
    z = xc / (xc.square().mean(-1, keepdim=True) + EPS).sqrt() * w
    z = z if b is None else z + b
    return z * torch.sigmoid(z) if silu else z


def _inputs(width, rows, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    draw = lambda: torch.randn(rows, width, generator=g) * torch.exp(0.3 * torch.randn(rows, 1, generator=g))  # noqa: E731
    return {"x": draw() + 0.5, "w": 1 + 0.2 * torch.randn(width, generator=g),
            "b": 0.3 * torch.randn(width, generator=g) if bias else None, "dy": draw(), "u": draw()}


def _leaves(d, device, dtype):
    return {k: None if v is None else v.to(device=device, dtype=dtype).requires_grad_() for k, v in d.items()}


def _all_orders(t, y):
    names = [k for k in ("x", "w", "b") if t[k] is not None]
    first = torch.autograd.grad(y, [t[k] for k in names], t["dy"], retain_graph=True)
    out = {"y": y, **{"d" + k: g for k, g in zip(names, first)}}
    again, = torch.autograd.grad(y, t["x"], t["dy"], create_graph=True)
    second = torch.autograd.grad(again, [t[k] for k in names] + [t["dy"]], t["u"].detach(), allow_unused=True)
    out.update({"dd" + k: g for k, g in zip(names + ["dy"], second)})
    return out


def _compare(got, want, rtol=1e-5):
    assert got.keys() == want.keys()
    for k, w in want.items():
        if w is None:
            assert got[k] is None or not got[k].any(), k
        else:
            assert got[k] is not None, k
            assert_rel(got[k], w, rtol=rtol, what=k)


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("width,rows", SHAPES)
def test_every_order(gpu, width, rows, silu):
    from ictc_o3.operators import layer_norm
    d = _inputs(width, rows, width * 7 + rows, bias=width % 3 != 1)
    t, r = _leaves(d, gpu, torch.float32), _leaves(d, "cpu", torch.float64)
    y = layer_norm(t["x"], t["w"], t["b"], eps=EPS, activation="silu" if silu else None)
    want = _all_orders(r, _formula(r["x"], r["w"], r["b"], silu))
    got = _all_orders(t, y)
    if width == 1:      # xh is zero, and so is every gradient to x; what 64 bits leave of it is no scale
        for k in ("dx", "ddx", "ddw", "dw", "dddy"):
            assert got.pop(k).abs().max() <= 1e-9 and want.pop(k).abs().max() <= 1e-9
        if "ddb" in got:
            a, b = got.pop("ddb"), want.pop("ddb")
            assert (a is None or a.abs().max() <= 1e-9) and (b is None or b.abs().max() <= 1e-9)
    _compare(got, want)


@pytest.mark.parametrize("silu", [False, True])
def test_gradients_against_differences(gpu, silu):
    """Directional derivatives of the kernels' first and second order against central differences in 64 bits."""
    from ictc_o3.operators import layer_norm
    d = _inputs(24, 6, 3)
    t, r = _leaves(d, gpu, torch.float32), {k: v.double() for k, v in d.items()}
    y = layer_norm(t["x"], t["w"], t["b"], eps=EPS, activation="silu" if silu else None)
    dx, = torch.autograd.grad(y, t["x"], t["dy"], create_graph=True)
    gx, gdy = torch.autograd.grad(dx, [t["x"], t["dy"]], t["u"].detach())
    v = torch.randn(6, 24, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    h = 1e-5

    def value(x):
        return (_formula(x, r["w"], r["b"], silu) * r["dy"]).sum()

    def slope(x, dy):
        x = x.clone().requires_grad_()
        g, = torch.autograd.grad(_formula(x, r["w"], r["b"], silu), x, dy)
        return (g * r["u"]).sum()

    # (central differences: h^2 of a third derivative of order 1 to 10, and 1e-16 / h of the values)
    near = dict(rel=1e-5, abs=1e-5)
    assert (dx.detach().double().cpu() * v).sum() == pytest.approx(
        ((value(r["x"] + h * v) - value(r["x"] - h * v)) / (2 * h)).item(), **near)
    assert (gx.double().cpu() * v).sum() == pytest.approx(
        ((slope(r["x"] + h * v, r["dy"]) - slope(r["x"] - h * v, r["dy"])) / (2 * h)).item(), rel=1e-5, abs=1e-4)
    assert (gdy.double().cpu() * v).sum() == pytest.approx(
        ((slope(r["x"], r["dy"] + h * v) - slope(r["x"], r["dy"] - h * v)) / (2 * h)).item(), **near)


@pytest.mark.parametrize("silu", [False, True])
def test_third_order_and_weight_cotangents(gpu, silu):
    """A gradient of second gradients, and cotangents of weight gradients: the composed formulas."""
    from ictc_o3.operators import layer_norm
    d = _inputs(20, 7, 11)
    results = []
    for t, f in ((_leaves(d, gpu, torch.float32),
                  lambda t: layer_norm(t["x"], t["w"], t["b"], eps=EPS, activation="silu" if silu else None)),
                 (_leaves(d, "cpu", torch.float64), lambda t: _formula(t["x"], t["w"], t["b"], silu))):
        dx, dw = torch.autograd.grad(f(t), [t["x"], t["w"]], t["dy"], create_graph=True)
        ddx, ddy = torch.autograd.grad((dx * t["u"]).sum() + (dw * t["w"].detach().flip(0)).sum(), [t["x"], t["dy"]],
                                       create_graph=True)
        results.append(dict(zip("xwyu", torch.autograd.grad((ddx * t["dy"].detach()).sum() + ddy.square().sum(),
                                                            [t["x"], t["w"], t["dy"], t["u"]]))))
    _compare(*results)


def test_large_means_and_single_entries(gpu):
    """Rows far from zero, with one large entry, or of two values: what is left of a cotangent is a small
    difference, which 64-bit statistics keep (float32 inputs are the same in the reference)."""
    from ictc_o3.operators import layer_norm
    for width in (2, 64, 300, 1500):
        d = _inputs(width, 12, width)
        d["x"][:4] += 3000.0
        d["x"][4:8, 0] = 500.0
        d["x"][8:10] = 2.5
        t, r = _leaves(d, gpu, torch.float32), _leaves(d, "cpu", torch.float64)
        got = _all_orders(t, layer_norm(t["x"], t["w"], t["b"], eps=EPS))
        want = _all_orders(r, _formula(r["x"], r["w"], r["b"], False))
        assert_rel(got["y"], want["y"], what="y")
        for rows in (slice(0, 4), slice(4, 8), slice(8, 10), slice(10, 12)):
            for k in ("dx", "ddx", "dddy"):      # each kind of row against its own scale
                if want[k][rows].abs().max() > 0:
                    assert_rel(got[k][rows], want[k][rows], rtol=2e-5, what=f"{width} {k} {rows}")


def test_infinities_and_nans_stay_in_their_rows(gpu):
    from ictc_o3.operators import layer_norm
    d = _inputs(70, 40, 5)
    clean = _leaves(d, gpu, torch.float32)
    d["x"][7, 3], d["x"][21, 69] = float("inf"), float("nan")
    t = _leaves(d, gpu, torch.float32)
    for silu in (None, "silu"):
        a, b = (layer_norm(s["x"], s["w"], s["b"], eps=EPS, activation=silu) for s in (t, clean))
        da, db = (torch.autograd.grad(y, s["x"], s["dy"])[0] for y, s in ((a, t), (b, clean)))
        rest = [i for i in range(40) if i not in (7, 21)]
        assert a[[7, 21]].isnan().all() and torch.equal(a[rest], b[rest]) and torch.equal(da[rest], db[rest])


@pytest.mark.parametrize("shape", [(0, 16), (3, 0, 8)])
def test_no_rows(gpu, shape):
    from ictc_o3.operators import layer_norm
    x = torch.empty(*shape, device=gpu, requires_grad=True)
    w, b = (torch.ones(shape[-1], device=gpu, requires_grad=True) for _ in range(2))
    y = layer_norm(x, w, b, activation="silu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y), create_graph=True)
    assert y.shape == x.shape and dx.shape == x.shape and not dw.any() and not db.any()
    gx, gw = torch.autograd.grad(dx, (x, w), torch.empty_like(dx))
    assert gx.shape == x.shape and not gw.any()


def test_leading_axes_strides_and_alignment(gpu):
    from ictc_o3.operators import layer_norm
    g = torch.Generator().manual_seed(2)
    flat = torch.randn(4 * 5 * 66 + 1, generator=g).to(gpu)
    x = flat[1:].view(4, 5, 66)                     # one float off any vector's alignment
    w, b = (torch.randn(67, generator=g).to(gpu)[1:] for _ in range(2))
    want = _formula(x.double().cpu(), w.double().cpu(), b.double().cpu(), True)
    assert_rel(layer_norm(x, w, b, activation="silu"), want)
    turned = torch.randn(5, 66, 4, generator=g).to(gpu).permute(2, 0, 1)
    assert not turned.is_contiguous()
    assert_rel(layer_norm(turned, w, b), _formula(turned.double().cpu(), w.double().cpu(), b.double().cpu(), False))
    dx, = torch.autograd.grad(layer_norm(turned.requires_grad_(), w, b), turned, torch.ones(1, device=gpu).expand(4, 5, 66))
    assert dx.shape == turned.shape


def test_partial_requirements(gpu):
    """Only the gradients that are asked for, with the same values as all of them."""
    from ictc_o3.operators import layer_norm
    t = _leaves(_inputs(48, 50, 9), gpu, torch.float32)
    full = torch.autograd.grad(layer_norm(t["x"], t["w"], t["b"], activation="silu"), [t["x"], t["w"], t["b"]], t["dy"])
    for k, want in zip("xwb", full):
        alone = {n: v.detach().requires_grad_(n == k) for n, v in t.items()}
        got, = torch.autograd.grad(layer_norm(alone["x"], alone["w"], alone["b"], activation="silu"), alone[k], t["dy"])
        assert torch.equal(got, want), k


def test_runs_agree_in_bits_and_on_another_stream(gpu):
    from ictc_o3.operators import layer_norm
    t = _leaves(_inputs(64, 30000, 1), gpu, torch.float32)
    results = []
    for k in range(2):
        stream = torch.cuda.Stream() if k else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            results.append(_all_orders(t, layer_norm(t["x"], t["w"], t["b"], activation="silu")))
        torch.cuda.synchronize()
    for k in results[0]:
        assert torch.equal(results[0][k], results[1][k]), k


def test_captured_passes(gpu):
    """Forward, gradients and second gradients in a graph, replayed on new inputs between eager calls."""
    from ictc_o3.operators import layer_norm
    t = _leaves(_inputs(64, 700, 21), gpu, torch.float32)

    def work(x, w, b, dy, u):
        x, dy = x.detach().requires_grad_(), dy.detach().requires_grad_()
        w, b = w.detach().requires_grad_(), b.detach().requires_grad_()
        y = layer_norm(x, w, b, activation="silu")
        dx, = torch.autograd.grad(y, x, dy, create_graph=True)
        return [y.detach(), dx.detach(), *torch.autograd.grad(dx, (x, w, b, dy), u)]

    static = {k: v.detach().clone() for k, v in t.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work(**static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(**static)
    for seed in range(3):
        new = _inputs(64, 700, 100 + seed)
        for k, v in static.items():
            v.copy_(new[k])
        graph.replay()
        want = work(**{k: v.clone() for k, v in static.items()})
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_refusals(gpu):
    from ictc_o3.operators import layer_norm
    x, w = torch.zeros(3, 8, device=gpu), torch.ones(8, device=gpu)
    for call in (lambda: layer_norm(x, w[:7]), lambda: layer_norm(x, w, w[:7]), lambda: layer_norm(x, w, eps=0.0),
                 lambda: layer_norm(x, w, eps=float("nan")), lambda: layer_norm(x, w, activation="gelu"),
                 lambda: layer_norm(x.double(), w.double()), lambda: layer_norm(x, w.cpu()),
                 lambda: layer_norm(x.half(), w.half()), lambda: layer_norm(x[0, 0], w),
                 lambda: layer_norm(torch.zeros(2, 8193, device=gpu), torch.ones(8193, device=gpu)),
                 lambda: layer_norm(torch.zeros(2, 0, device=gpu), torch.ones(0, device=gpu))):
        with pytest.raises(ValueError):
            call()
    with torch.autocast("cuda"), pytest.raises(ValueError):
        layer_norm(x, w)


def test_inference_and_no_grad(gpu):
    from ictc_o3.operators import layer_norm
    t = _leaves(_inputs(64, 30, 6), gpu, torch.float32)
    want = layer_norm(t["x"], t["w"], t["b"])
    with torch.no_grad():
        assert torch.equal(layer_norm(t["x"], t["w"], t["b"]), want.detach())
    with torch.inference_mode():
        fresh = t["x"].clone()
        assert torch.equal(layer_norm(fresh, t["w"], t["b"]), want)
    assert want.requires_grad


def test_two_streams_at_once(gpu):
    """Passes side by side have workspaces of their own."""
    from ictc_o3.operators import layer_norm
    cases = [_leaves(_inputs(64, 40000, 30 + k), gpu, torch.float32) for k in range(2)]

    def work(t):
        return torch.autograd.grad(layer_norm(t["x"], t["w"], t["b"], activation="silu"), [t["x"], t["w"], t["b"]], t["dy"])

    want = [[g.clone() for g in work(t)] for t in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, t in zip(streams, cases):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(work(t))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_changed_inputs_are_noticed(gpu):
    """An input that was changed in place after the forward pass is refused by the backward pass."""
    from ictc_o3.operators import layer_norm
    t = _leaves(_inputs(16, 5, 2), gpu, torch.float32)
    x = t["x"].detach().clone().requires_grad_()
    held = x * 1.0
    y = layer_norm(held, t["w"], t["b"])
    with torch.no_grad():
        held.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, x, t["dy"])
