"""Orthogonalised updates against plain float64 iterations on the CPU: matrices of every kind of size, rank-deficient
and badly scaled ones, the optimizer's step, clipping, empty and missing tensors, graphs, streams and refusals.

Tolerances.  Operands are kept to 22 bits and products are summed in float32: relative errors of about 2^-22 (and
sqrt(K) 2^-24 for sums of K terms) of the largest singular value in each of three products a step.  A step multiplies
errors of small singular values, like those themselves, by up to 3.4 (a), those near 1 by at most |p'| = 2: five steps
grow the first one's error by 3.4^5 = 485 of a singular value that is then below 1, and later ones by less.
sum_k 3 * 3.4^k * 2^-22 = 5e-4 would be reached if every singular value were tiny and every error in phase; errors of
independent entries spread over the directions, 1 / sqrt(m) each, and only the small ones' share grows: 1e-5 of the
result's 2-norm at random matrices, 3e-5 at rank-deficient ones, which is what the comparison below allows
(float32 iterations themselves reach 1e-6 to 2e-5)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
SHAPES = [(1, 1), (1, 77), (77, 1), (2, 3), (5, 5), (16, 17), (31, 33), (32, 32), (63, 65), (64, 64), (65, 64), (64, 8),
          (100, 41), (127, 129), (128, 128), (129, 130), (128, 700), (700, 128), (64, 3000), (2500, 40), (300, 257),
          (513, 511), (1024, 200), (3, 64, 64), (2, 3, 20, 30), (1, 5, 7), (4, 130, 64), (150, 12, 9)]


def _exact(u, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = u.double().cpu()
    x = x.reshape(-1, *x.shape[-2:])
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + eps)
    turned = x.shape[1] > x.shape[2]
    x = x.mT if turned else x
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    return (x.mT if turned else x).reshape(u.shape)


def _check(got, want, tolerance=1e-5, what=""):
    assert got.shape == want.shape and got.dtype == torch.float32 and got.is_contiguous()
    error, size = (got.double().cpu() - want).norm(), want.norm()
    assert error <= tolerance * size, (what, (error / size).item())


def _draw(shape, seed, scale=1.0):
    return scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_one_shape(gpu, shape):
    from ictc_o3.operators import orthogonalize
    u = _draw(shape, sum(shape))
    got, = orthogonalize([u.to(gpu)])
    _check(got, _exact(u))


def test_all_shapes_together(gpu):
    from ictc_o3.operators import orthogonalize
    us = [_draw(s, k, 10.0 ** (k % 7 - 3)) for k, s in enumerate(SHAPES * 5)]      # more than a launch's table holds
    got = orthogonalize([u.to(gpu) for u in us])
    assert len(got) == len(us)
    for u, g in zip(us, got):
        _check(g, _exact(u), what=tuple(u.shape))


@pytest.mark.parametrize("shape", [(60, 64), (128, 128), (200, 90), (600, 520)])
def test_rank_deficient(gpu, shape):
    """Singular values over six orders, a quarter of them zero: those that stay far below 1 keep their digits too."""
    from ictc_o3.operators import orthogonalize
    k = min(shape)
    q, _ = torch.linalg.qr(_draw((shape[0], k), 1).double())
    r, _ = torch.linalg.qr(_draw((shape[1], k), 2).double())
    s = torch.logspace(0, -6, k, dtype=torch.float64)
    s[3 * k // 4:] = 0.0
    u = ((q * s) @ r.T).float()
    got, = orthogonalize([u.to(gpu)])
    _check(got, _exact(u), 3e-5)


def test_scales_steps_and_coefficients(gpu):
    """Norms from below eps to far above float32's squares; other polynomials and numbers of steps."""
    from ictc_o3.operators import orthogonalize
    for scale in (1e-30, 1e-9, 1e-7, 1.0, 1e18, 1e30):
        u = _draw((48, 80), 3, scale)
        got, = orthogonalize([u.to(gpu)])
        _check(got, _exact(u), what=scale)
    u = _draw((70, 50), 4)
    for steps in (1, 2, 3, 10):
        got, = orthogonalize([u.to(gpu)], steps=steps, coefficients=(1.875, -1.25, 0.375))
        _check(got, _exact(u, steps, (1.875, -1.25, 0.375)), what=steps)
    got, = orthogonalize([u.to(gpu)], eps=0.5)
    _check(got, _exact(u, eps=0.5))


def test_zeros_and_values_that_are_not_finite(gpu):
    """A matrix of zeros stays one; not-a-number stays in its matrix."""
    from ictc_o3.operators import orthogonalize
    us = [torch.zeros(40, 50), _draw((40, 50), 5), _draw((3, 70, 70), 6)]
    us[2][1, 4, 4] = float("nan")
    got = orthogonalize([u.to(gpu) for u in us])
    assert not got[0].any()
    _check(got[1], _exact(us[1]))
    assert got[2][1].isnan().all()
    _check(got[2][::2].contiguous(), _exact(us[2][::2]))


def test_empty_strided_and_unaligned(gpu):
    from ictc_o3.operators import orthogonalize
    assert orthogonalize([]) == []
    empty = [torch.empty(0, 5, device=gpu), torch.empty(3, 0, 4, device=gpu), torch.empty(5, 0, device=gpu)]
    assert [g.shape for g in orthogonalize(empty)] == [e.shape for e in empty]
    flat = torch.randn(33 * 47 + 1, device=gpu)
    odd, turned = flat[1:].view(33, 47), torch.randn(90, 66, device=gpu).t()
    got = orthogonalize([odd, empty[0], turned])
    _check(got[0], _exact(odd))
    _check(got[2], _exact(turned))


def _reference_step(p, g, m, *, lr, beta, nesterov, weight_decay, adjust, coefficient=1.0):
    p, g, m = p.double(), g.double() * coefficient, m.double()
    m = beta * m + (1 - beta) * g
    u = beta * m + (1 - beta) * g if nesterov else m
    r, c = p.shape[-2:]
    s = max(1.0, r / c) ** 0.5 if adjust == "original" else 0.2 * max(r, c) ** 0.5
    return (1 - lr * weight_decay) * p - lr * s * _exact(u), m


@pytest.mark.parametrize("nesterov,adjust,clipped,tensor_lr", [(True, "original", False, False),
                                                              (False, "match_rms_adamw", True, True)])
def test_step(gpu, nesterov, adjust, clipped, tensor_lr):
    from ictc_o3.operators import gradient_norm, muon_step
    shapes = [(64, 64), (7, 90), (200, 30), (3, 32, 32), (129, 300), (1, 1)]
    ps, gs, ms = ([_draw(s, 10 * j + k, scale) for k, s in enumerate(shapes)]
                  for j, scale in ((1, 0.1), (2, 1e-2), (3, 5e-3)))
    own = [[t.to(gpu) for t in ts] for ts in (ps, gs, ms)]
    grads = list(own[1])
    grads[2] = None
    clip = gradient_norm(grads, 0.3) if clipped else None
    options = dict(beta=0.9, nesterov=nesterov, weight_decay=0.05, adjust=adjust)
    versions = [t._version for t in own[0] + own[2]]
    muon_step(own[0], grads, own[2], lr=torch.tensor([0.02], device=gpu) if tensor_lr else 0.02, clip=clip, **options)
    coefficient = 1.0 if clip is None else clip[1].item()
    assert not clipped or 0.0 < coefficient < 1.0
    for k, (p, g, m) in enumerate(zip(ps, gs, ms)):
        if k == 2:
            assert torch.equal(own[0][k].cpu(), p) and torch.equal(own[2][k].cpu(), m)
            continue
        want_p, want_m = _reference_step(p, g, m, lr=0.02, coefficient=coefficient, **options)
        # the update to 1e-5 of itself, and a rounding of the sum (the float32 step's constants: 2^-24 each)
        error = (own[0][k].double().cpu() - want_p).norm()
        assert error <= 1e-5 * (want_p - p.double()).norm() + 2e-7 * want_p.norm()
        assert (own[2][k].double().cpu() - want_m).norm() <= 2e-7 * want_m.norm()
    raised = [t._version > v for t, v in zip(own[0] + own[2], versions)]
    assert raised == [k % 6 != 2 for k in range(12)]


def test_a_norm_that_is_not_finite_changes_nothing(gpu):
    from ictc_o3.operators import gradient_norm, muon_step
    p, g, m = (_draw((50, 50), k).to(gpu) for k in range(3))
    g[3, 3] = float("inf")
    before = p.clone(), m.clone()
    muon_step([p], [g], [m], lr=0.1, clip=gradient_norm([g], 1.0))
    assert torch.equal(p, before[0]) and torch.equal(m, before[1])


def test_unaligned_parameters_and_strided_gradients(gpu):
    from ictc_o3.operators import muon_step
    flat = torch.randn(3 * (45 * 31 + 1), device=gpu).mul_(0.1)
    p, m = flat[1:1 + 45 * 31].view(45, 31), flat[1500 + 1:1500 + 1 + 45 * 31].view(45, 31)
    g = torch.randn(31, 45, device=gpu).t()
    want_p, _ = _reference_step(p.cpu(), g.cpu(), m.cpu(), lr=0.5, beta=0.95, nesterov=True, weight_decay=0.0,
                                adjust="original")
    rest = flat.clone()
    muon_step([p], [g], [m], lr=0.5)
    _check(p.contiguous(), want_p)
    changed = (flat != rest).nonzero().flatten()
    inside = ((changed >= 1) & (changed < 1 + 45 * 31)) | ((changed >= 1501) & (changed < 1501 + 45 * 31))
    assert bool(inside.all())


def test_runs_agree_in_bits_in_any_company_and_on_another_stream(gpu):
    from ictc_o3.operators import orthogonalize
    us = [_draw(s, k).to(gpu) for k, s in enumerate([(64, 300), (130, 130), (512, 200), (9, 9)])]
    first = orthogonalize(us)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = orthogonalize(us)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_captured_orthogonalisation(gpu):
    from ictc_o3.operators import orthogonalize
    static = [_draw(s, k).to(gpu) for k, s in enumerate([(64, 64), (128, 300), (200, 90)])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        orthogonalize(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(static)
    for seed in range(3):
        for k, t in enumerate(static):
            t.copy_(_draw(t.shape, 40 + 10 * seed + k))
        graph.replay()
        want = orthogonalize([t.clone() for t in static])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_more_than_one_group(gpu):
    """Workspaces of large calls are those of their largest group: results are the same as alone."""
    from ictc_o3.operators import orthogonalize
    big = [torch.randn(2100, 16000, device=gpu) for _ in range(6)]        # 0.4 GB of workspace each
    both = orthogonalize(big + [big[0][:50, :60].contiguous()])
    alone, = orthogonalize([big[5]])
    assert torch.equal(both[5], alone)
    _check(both[6], _exact(big[0][:50, :60]))
    gram = both[5].double() @ both[5].double().T
    values = torch.linalg.eigvalsh(gram)
    assert 0.4 < values.min() and values.max() < 1.6


def test_refusals(gpu):
    from ictc_o3.operators import muon_step, orthogonalize
    x = torch.randn(4, 4, device=gpu)
    for call in (lambda: orthogonalize([x[0]]), lambda: orthogonalize([x.double()]), lambda: orthogonalize([x.cpu()]),
                 lambda: orthogonalize([x], steps=0), lambda: orthogonalize([x], steps=65),
                 lambda: orthogonalize([x], steps=2.0), lambda: orthogonalize([x], eps=0.0),
                 lambda: orthogonalize([x], eps=float("nan")), lambda: orthogonalize([x], coefficients=(1.0, 2.0)),
                 lambda: orthogonalize([x], coefficients=(1.0, 2.0, float("inf"))), lambda: orthogonalize([None])):
        with pytest.raises(ValueError):
            call()
    p, g, m = (x.clone() for _ in range(3))
    step = lambda *a, **k: muon_step(*a, **{"lr": 0.1, **k})     # noqa: E731
    for call in (lambda: step([p], [g], [m[:2]]), lambda: step([p], [g], []), lambda: step([p], [g[:2]], [m]),
                 lambda: step([p], [g], [m.t()]), lambda: step([p.t()], [g], [m]), lambda: step([p[0]], [g[0]], [m[0]]),
                 lambda: step([p], [g], [m], lr=-1.0), lambda: step([p], [g], [m], beta=1.0),
                 lambda: step([p], [g], [m], weight_decay=-0.1), lambda: step([p], [g], [m], adjust="none"),
                 lambda: step([p], [g], [m], lr=torch.ones(2, device=gpu)), lambda: step([p], [g], [m], clip=x[0]),
                 lambda: step([], [], [])):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(p, x) and torch.equal(m, x)


def test_two_streams_at_once(gpu):
    from ictc_o3.operators import orthogonalize
    cases = [[_draw(s, k).to(gpu) for k, s in enumerate(shapes)]
             for shapes in ([(64, 900), (128, 128), (30, 30)], [(300, 700), (90, 400)])]
    want = [[x.clone() for x in orthogonalize(c)] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, c in zip(streams, cases):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(orthogonalize(c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_in_place_and_the_same_matrix_twice(gpu):
    """What reads a matrix twice may; a captured step's moving averages go on from replay to replay."""
    from ictc_o3.operators import muon_step, orthogonalize
    u = _draw((70, 90), 1).to(gpu)
    a, b = orthogonalize([u, u])
    assert torch.equal(a, b)
    p, m = _draw((70, 90), 2).to(gpu), torch.zeros(70, 90, device=gpu)
    q, n = p.clone(), m.clone()
    rate = torch.tensor([0.1], device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        muon_step([p], [u], [m], lr=rate)
        muon_step([q], [u], [n], lr=rate)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step([p], [u], [m], lr=rate)
    for k in range(3):
        u.copy_(_draw((70, 90), 10 + k))
        rate.fill_(0.1 / (k + 1))
        graph.replay()
        muon_step([q], [u.clone()], [n], lr=0.1 / (k + 1))
        torch.cuda.synchronize()
        # (the rate as a float32 tensor and as a number: the same bits)
        assert torch.equal(p, q) and torch.equal(m, n)


def test_coefficients_beyond_the_range(gpu):
    """Singular values that grow without bound are seen as such."""
    from ictc_o3.operators import orthogonalize
    got, other = orthogonalize([_draw((40, 40), 3).to(gpu), torch.zeros(8, 8, device=gpu)], steps=8, coefficients=(4.0, 0.0, 0.0))
    assert not got.isfinite().all() and not other.any()


def test_both_kinds_of_matrices_captured(gpu):
    """Matrices with short and with long shorter sides, which run on two streams, in a graph; and in between them
    eager calls on another stream."""
    from ictc_o3.operators import muon_step
    shapes = [(40, 300), (200, 300), (3, 64, 64), (150, 150)]
    first = [[_draw(s, 10 * j + k, scale).to(gpu) for k, s in enumerate(shapes)] for j, scale in ((1, 0.1), (2, 0.01), (3, 0.0))]
    second = [[t.clone() for t in ts] for ts in first]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        muon_step(*first, lr=0.1)
        muon_step(*second, lr=0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step(*first, lr=0.1)
    for seed in range(3):
        for k, (g, h) in enumerate(zip(first[1], second[1])):
            g.copy_(_draw(g.shape, 100 * seed + k, 0.01))
            h.copy_(g)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            muon_step(*second, lr=0.1)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(first, second) for a, b in zip(x, y))


def test_written_memory_that_overlaps_is_refused(gpu):
    from ictc_o3.operators import muon_step
    flat = _draw((8, 20), 5).to(gpu)
    kept = flat.clone()
    p, q, m, n = flat[:2], flat[2:4], flat[4:6], flat[6:]      # side by side
    g = _draw((2, 20), 6).to(gpu)
    for params, grads, momentum in (([p, p], [g, g], [m, q]), ([p, flat[1:3]], [g, g], [m, flat[4:6]]), ([p], [g], [p]),
                                    ([p, q], [g, g], [m, m]), ([p], [p], [m]), ([p], [m], [m]),
                                    ([p, q], [g, flat[1:3]], [m, flat[5:7]])):
        with pytest.raises(ValueError, match="overlap"):
            muon_step(params, grads, momentum, lr=0.1)
    assert torch.equal(flat, kept)
    muon_step([p, p, q], [g, None, g], [m, m, n[:2]], lr=0.1)  # without a gradient nothing is written; gradients may be one
    assert not any(torch.equal(a, b) for a, b in zip(flat.split(2), kept.split(2)))
