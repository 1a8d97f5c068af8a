"""The AdamW step over many tensors and the gradient norm against plain float64 formulas.

u = 2^-24 is float32's unit roundoff.  A moment is two products and a sum of operands that are
themselves rounded (the decay factors, the clipped gradient): within 6 u of |b1 m| + |(1 - b1) c g|.
The update adds the rounding of two quotients, a root and the bias corrections (each in float32: 1 u)
to the first moment's error: 16 u of the update formed from |b1 m| + |(1 - b1) c g|; the parameter's own
product and sum: 3 u of |p|.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LR, BETAS, EPS, DECAY = 3e-3, (0.9, 0.999), 1e-8, 0.02

# single values, block ends on either side, more tensors than one launch takes, a large one
SIZES = {"one": [1], "ends": [255, 256, 257, 1023, 1024, 1025, 0, 3], "many": [1 + 37 * k % 700 for k in range(331)],
         "large": [3_000_001, 5, 70_000]}


def _inputs(sizes, seed, gpu, offset=0):
    """Parameters and gradients (views `offset` floats into their buffers) with scales of their own."""
    gen = torch.Generator().manual_seed(seed)
    params, grads = [], []
    for k, n in enumerate(sizes):
        level = 10.0 ** (-3 + k % 4)
        params.append((torch.randn(n + offset, generator=gen) * 0.1).to(gpu)[offset:])
        grads.append((torch.randn(n + offset, generator=gen) * torch.exp(torch.randn(n + offset, generator=gen))
                      * level).to(gpu)[offset:])
    return params, grads


def _starts(sizes):
    return np.concatenate([[0], np.cumsum([-(-n // 256) * 256 for n in sizes])]).astype(np.int64)


def _mix(x):
    x = x.astype(np.uint32)
    x ^= x >> np.uint32(16)
    x *= np.uint32(0xBB67AE85)
    x ^= x >> np.uint32(15)
    x *= np.uint32(0x6A09E667)
    return x ^ (x >> np.uint32(16))


def _decode(codes, top, mantissa_low):
    """8-bit codes (magnitudes) as float64; mantissa_low: exponent of the step of code 1 (block exponent 0)."""
    field = codes >> 3
    return ((codes & 7) + 8 * (field > 0)) * np.exp2(np.maximum(field, 1) + float(mantissa_low)) \
        * np.repeat(np.exp2(top.astype(np.float64) - 127), 256)


def _values(m, v):
    """The float64 values of 8-bit moments ((codes, exponents) pairs of numpy arrays)."""
    mc, vc = m[0].astype(np.int64), v[0].astype(np.int64)
    return _decode(mc & 127, m[1], -18) * np.where(mc > 127, -1.0, 1.0), _decode(vc, v[1], -34)


def _formula(p, g, m, v, steps, coefficient=1.0, lr=LR):
    """(p, m, v) after the step and what their tolerances go by."""
    b1, b2 = BETAS
    g = g * coefficient
    new_m, new_v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    denom = np.sqrt(new_v / (1 - b2 ** steps)) + EPS
    rate = lr / (1 - b1 ** steps)
    size_m = np.abs(b1 * m) + np.abs((1 - b1) * g)
    return ((1 - lr * DECAY) * p - rate * new_m / denom, new_m, new_v,
            U * (3 * np.abs(p) + 16 * rate * size_m / denom), 6 * U * size_m, 8 * U * new_v)


def _host(tensors):
    return [t.detach().cpu().double().numpy() for t in tensors]


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("name", list(SIZES))
def test_steps_match_the_formula(gpu, name, offset):
    from ictc_o3.backends.hip.optimizer import adamw_step, gradient_norm, new_state
    sizes = SIZES[name]
    params, grads = _inputs(sizes, 1, gpu, offset)
    state = new_state(params)
    at = _starts(sizes)
    for step in range(1, 4):
        _, grads = _inputs(sizes, 10 + step, gpu, offset)
        before_p, before_g = _host(params), _host(grads)
        before_m, before_v = _host(state[:2])
        clip = gradient_norm(grads, 0.5) if step == 2 else None
        coefficient = 1.0
        if clip is not None:
            norm = math.sqrt(sum(float((g * g).sum()) for g in before_g))
            coefficient = min(1.0, 0.5 / norm)
            got = clip.cpu().double().numpy()
            np.testing.assert_allclose(got, [norm, coefficient], rtol=2 * U)
        adamw_step(params, grads, *state, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, clip=clip)
        torch.cuda.synchronize()
        m, v = _host(state[:2])
        for k, (p, n) in enumerate(zip(_host(params), sizes)):
            s = slice(at[k], at[k] + n)
            want = _formula(before_p[k], before_g[k], before_m[s], before_v[s], step, coefficient)
            for got, value, tol in zip((p, m[s], v[s]), want[:3], want[3:]):
                assert np.all(np.abs(got - value) <= tol), (k, n, np.max(np.abs(got - value) - tol))
            assert not m[at[k] + n:at[k + 1]].any() and not v[at[k] + n:at[k + 1]].any()
        progress = state[2].cpu().numpy()
        np.testing.assert_allclose(progress, [[step, BETAS[0] ** step, BETAS[1] ** step]] * len(sizes), rtol=1e-14)


@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("name", list(SIZES))
def test_eight_bit_steps(gpu, name, offset):
    """Codes, exponents and parameters of three steps from the stored values before each: rounding
    follows the documented hash, and a code may differ from float64's only where the value plus its
    random offset lies within the float32 error of a whole step."""
    from ictc_o3.backends.hip.optimizer import adamw_step, moment_values, new_state
    sizes, seed = SIZES[name], 77
    params, _ = _inputs(sizes, 2, gpu, offset)
    state = new_state(params, 8)
    at = _starts(sizes)
    total = int(at[-1])
    for step in range(1, 4):
        _, grads = _inputs(sizes, 20 + step, gpu, offset)
        before_p, before_g = _host(params), _host(grads)
        old = [(c.cpu().numpy(), t.cpu().numpy()) for c, t in state[:2]]
        old_m, old_v = _values(*old)
        adamw_step(params, grads, *state, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, seed=seed)
        torch.cuda.synchronize()
        new = [(c.cpu().numpy(), t.cpu().numpy()) for c, t in state[:2]]
        got_m, got_v = _values(*new)
        m, v, tol_m, tol_v = (np.zeros(total) for _ in range(4))
        for k, (p, n) in enumerate(zip(_host(params), sizes)):
            s = slice(at[k], at[k] + n)
            want = _formula(before_p[k], before_g[k], old_m[s], old_v[s], step)
            assert np.all(np.abs(p - want[0]) <= want[3]), (k, n)
            m[s], v[s], tol_m[s], tol_v[s] = want[1], want[2], want[4], want[5]
        with np.errstate(over="ignore"):
            key = _mix(np.array([(seed + step * 0x9E3779B9) & 0xFFFFFFFF], dtype=np.uint64))
            bits = _mix(np.arange(total, dtype=np.uint32) + key)
        for x, tol, got, top, lowest, raw in ((m, tol_m, got_m, new[0][1], -14, bits & 0xFFFF),
                                              (v, tol_v, got_v, new[1][1], -30, bits >> 16)):
            largest = np.abs(x).reshape(-1, 256).max(1)
            mantissa, e = np.frexp(largest)
            want_top = np.maximum(np.where(mantissa > 0.875, e + 1, e) + 126, 1)
            near = np.abs(mantissa - 0.875) < 16 * U       # the raise decided by the last bits
            assert np.all((top == want_top) | near | (largest == 0))
            unit = np.exp2(np.maximum(np.frexp(np.abs(x))[1] - 1, np.repeat(top.astype(int) - 127, 256) + lowest) - 3.0)
            q = np.abs(x) / unit + raw / 65536.0
            value = np.floor(q) * unit * np.sign(x)
            if lowest == -30:
                value = np.where((value == 0) & (x > 0), unit, value)
            unsure = np.abs(q - np.round(q)) <= tol / unit + 16 * U
            assert np.all((got == value) | unsure), np.flatnonzero((got != value) & ~unsure)[:5]
            assert np.all(np.abs(got - value) <= np.where(unsure, unit * (1 + 1e-9), 0))
            assert np.all(got[x > 0] > 0) if lowest == -30 else True
        for values, want in zip(moment_values(*state[:2]), (got_m, got_v)):
            assert np.array_equal(values.double().cpu().numpy(), want)


def test_eight_bit_averages_are_kept(gpu):
    """Constant gradients for 800 steps: v tends to (1 - b2^t) g^2 on average (a rounding to the nearest
    code would leave it near its value after some ten steps).  One element's relative deviation is at most about
    0.5 (the step's p (1 - p) unit^2 summed over the average's memory), so the mean over 64 blocks has a
    standard deviation below 0.5 / 128: five of them are allowed."""
    from ictc_o3.backends.hip.optimizer import adamw_step, moment_values, new_state
    n = 64 * 256
    gen = torch.Generator().manual_seed(3)
    g = (torch.randn(n, generator=gen) + 3.0).abs().clamp(min=0.5).to(gpu)
    p = torch.zeros(n, device=gpu)
    state = new_state([p], 8)
    for _ in range(800):
        adamw_step([p], [g], *state, lr=0.0, betas=BETAS)
    m, v = moment_values(*state[:2])
    assert abs(float((v.double() / g.double() ** 2).mean()) / (1 - BETAS[1] ** 800) - 1) <= 5 * 0.5 / 128
    assert abs(float((m.double() / g.double()).mean()) - 1) <= 5 * 0.5 / 128


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-12, 1e-3])
def test_small_gradients_and_other_eps(gpu, bits, eps):
    """Gradients far below the usual eps, on either side of where the 8-bit kernel takes approximate roots."""
    from ictc_o3.backends.hip.optimizer import adamw_step, new_state
    params, grads = _inputs([700, 64], 11, gpu)
    grads = [g * 1e-10 for g in grads]
    state = new_state(params, bits)
    before, values = _host(params), _host(grads)
    adamw_step(params, grads, *state, lr=LR, betas=BETAS, eps=eps, weight_decay=DECAY)
    for p, old, g in zip(_host(params), before, values):
        m, v = (1 - BETAS[0]) * g, (1 - BETAS[1]) * g * g
        denom = np.sqrt(v / (1 - BETAS[1])) + eps
        rate = LR / (1 - BETAS[0])
        want = (1 - LR * DECAY) * old - rate * m / denom
        assert np.all(np.abs(p - want) <= U * (3 * np.abs(old) + 16 * rate * np.abs(m) / denom))


def test_a_tensor_without_a_gradient_keeps_its_state(gpu):
    from ictc_o3.backends.hip.optimizer import adamw_step, new_state
    sizes = [300, 5, 700]
    for bits in (32, 8):
        params, grads = _inputs(sizes, 4, gpu)
        state = new_state(params, bits)
        adamw_step(params, grads, *state, lr=LR)
        kept = params[1].clone()
        before = [t.clone() for part in state for t in ((part,) if isinstance(part, torch.Tensor) else part)]
        adamw_step(params, [grads[0], None, grads[2]], *state, lr=LR)
        after = [t for part in state for t in ((part,) if isinstance(part, torch.Tensor) else part)]
        assert torch.equal(params[1], kept)
        assert state[2][:, 0].tolist() == [2.0, 1.0, 2.0]
        for a, b in zip(after[:-1], before[:-1]):
            s = slice(512, 768) if a.numel() == 512 + 256 + 768 else slice(2, 3)
            assert torch.equal(a[s], b[s])


@pytest.mark.parametrize("bits", [32, 8])
def test_large_tensors_without_gradients(gpu, bits):
    """Tensors that end a launch because they take no part: the ones around them as in steps of their own."""
    from ictc_o3.backends.hip.optimizer import adamw_step, moment_values, new_state
    sizes = [300, 1_500_000, 700, 5, 1_200_000, 2_000_000, 40]
    params, grads = _inputs(sizes, 12, gpu)
    for k in (1, 4, 5):
        grads[k] = None
    before = [p.clone() for p in params]
    state = new_state(params, bits)
    adamw_step(params, grads, *state, lr=LR, seed=3)
    at = _starts(sizes)
    m, v = state[:2] if bits == 32 else moment_values(*state[:2])
    for k, g in enumerate(grads):
        part = slice(int(at[k]), int(at[k]) + sizes[k])
        if g is None:
            assert torch.equal(params[k], before[k]) and not m[part].any() and not v[part].any()
            continue
        alone, own = [before[k].clone()], new_state([before[k]], bits)
        adamw_step(alone, [g], *own, lr=LR, seed=3)
        assert torch.equal(params[k], alone[0])           # (a first step's update does not see the rounding)
        # 8-bit moments are rounded by their place in the state: within one code step of 1/8
        for got, want in zip((m, v), own[:2] if bits == 32 else moment_values(*own[:2])):
            exact = dict(rtol=0, atol=0) if bits == 32 else dict(rtol=0.125, atol=1e-4)
            torch.testing.assert_close(got[part], want[:sizes[k]], **exact)
    assert state[2][:, 0].tolist() == [1.0, 0.0, 1.0, 1.0, 0.0, 0.0, 1.0]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite(gpu, bits, bad):
    """Unclipped they go where the formula takes them and nowhere else; with the norm taken, the whole step is left out."""
    from ictc_o3.backends.hip.optimizer import adamw_step, gradient_norm, moment_values, new_state
    params, grads = _inputs([600], 5, gpu)
    state = new_state(params, bits)
    adamw_step(params, grads, *state, lr=LR)
    grads[0][300] = bad
    before = [params[0].clone(), state[2].clone()]
    clip = gradient_norm(grads, 1.0)
    assert math.isnan(clip[1].item()) and not math.isfinite(clip[0].item())
    adamw_step(params, grads, *state, lr=LR, clip=clip)
    assert torch.equal(params[0], before[0]) and torch.equal(state[2], before[1])
    adamw_step(params, grads, *state, lr=LR)
    m, v = state[:2] if bits == 32 else moment_values(*state[:2])
    broken = torch.zeros(768, dtype=torch.bool)
    broken[300] = True
    assert torch.equal(~torch.isfinite(m).cpu(), broken) and torch.equal(~torch.isfinite(v).cpu(), broken)
    assert torch.equal(~torch.isfinite(params[0]).cpu(), broken[:600])
    assert float(state[2][0, 0]) == 2.0


def test_gradient_norm_range_and_order(gpu):
    """Squares that overflow or vanish in float32, the same bits from run to run, None entries and zeros."""
    from ictc_o3.backends.hip.optimizer import gradient_norm
    for scale in (1e30, 1e-30, 1.0):
        _, grads = _inputs([7, 4096 * 3 + 1, 200_000], 6, gpu)
        grads = [g * scale for g in grads]
        want = math.sqrt(sum(float((g * g).sum()) for g in _host(grads)))
        a, b = gradient_norm([*grads, None], 2.0), gradient_norm([None, *grads], 2.0)
        assert torch.equal(a, b)
        np.testing.assert_allclose(a.cpu().double().numpy(), [want, min(1.0, 2.0 / want)], rtol=2 * U)
        assert gradient_norm(grads)[1].item() == 1.0
    zero = gradient_norm([torch.zeros(10, device=gpu), torch.zeros(0, device=gpu)], 1.0)
    assert zero.tolist() == [0.0, 1.0]


def test_optimizer_groups_state_and_versions(gpu):
    """Two groups, one clipped norm over both, a saved state that goes on bit for bit, a learning rate on the
    device, and version counters that show the change (caches of derived weights go by them)."""
    from ictc_o3.optim import AdamW
    for bits in (32, 8):
        def make():
            params, _ = _inputs([500, 33, 1200], 7, gpu)
            params = [torch.nn.Parameter(p.clone()) for p in params]
            return params, AdamW([{"params": params[:2], "lr": 1e-2}, {"params": params[2:], "weight_decay": 0.0}],
                                 lr=torch.tensor(1e-3, device=gpu), moment_bits=bits, max_grad_norm=0.3, seed=9)

        def steps(params, opt, first, count):
            for k in range(first, first + count):
                for p, g in zip(params, _inputs([500, 33, 1200], 30 + k, gpu)[1]):
                    p.grad = g
                opt.step()

        params, opt = make()
        version = params[0]._version
        steps(params, opt, 0, 2)
        assert params[0]._version > version
        norm = math.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in params))
        assert abs(opt.grad_norm[0].item() / norm - 1) <= 2 * U
        saved = {k: v for k, v in opt.state_dict().items()}
        other, opt2 = make()
        opt2.load_state_dict(saved)
        with torch.no_grad():
            for a, b in zip(other, params):
                a.copy_(b)
        steps(params, opt, 2, 2)
        steps(other, opt2, 2, 2)
        for a, b in zip(params, other):
            assert torch.equal(a, b)
        assert float(opt2.moments(other[2])[2]) == 4.0
        assert opt2.moments(other[1])[0].shape == other[1].shape


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays(gpu, bits):
    from ictc_o3.optim import AdamW
    from mace_hip import CapturedTrainingStep, training_step
    from test_mace_gpu import _setup
    from conftest import assert_rel
    model_a, graph, _, _ = _setup(gpu, atoms=64)
    model_b, _, _, _ = _setup(gpu, atoms=64)
    make = lambda model: AdamW(model.parameters(), lr=1e-3, moment_bits=bits, max_grad_norm=5.0)   # noqa: E731
    opt_a, opt_b = make(model_a), make(model_b)
    for _ in range(3):
        training_step(model_a, opt_a, dict(graph))
    captured = CapturedTrainingStep(model_b, opt_b, graph, warmup=3)
    for step in range(3):
        gen = torch.Generator(device=gpu).manual_seed(100 + step)
        pos = graph["positions"] + 0.05 * torch.randn(graph["positions"].shape, device=gpu, generator=gen)
        loss_a = training_step(model_a, opt_a, dict(graph, positions=pos))
        torch.cuda.synchronize(gpu)
        loss_b = captured(pos)
        torch.cuda.synchronize(gpu)
        assert_rel(loss_b, loss_a, rtol=1e-4, what=f"replay {step} loss")
    for a, b in zip(model_a.parameters(), model_b.parameters()):
        assert_rel(b, a, rtol=1e-4, what="parameter")


def test_refusals(gpu):
    from ictc_o3.backends.hip.optimizer import adamw_step, gradient_norm, moment_values, new_state
    from ictc_o3.optim import AdamW
    p, g = torch.zeros(300, device=gpu), torch.ones(300, device=gpu)
    m, v, progress = new_state([p])
    ok = dict(lr=1e-3)
    adamw_step([p], [g], m, v, progress, **ok)
    for args, more in ((([p], [g[:5]], m, v, progress), ok), (([p], [], m, v, progress), ok),
                       (([p], [g.double()], m, v, progress), ok), (([p.cpu()], [g], m, v, progress), ok),
                       (([p.view(20, 15).t()], [g.view(20, 15).t()], m, v, progress), ok),
                       (([p], [g], m[:256], v, progress), ok), (([p], [g], m, v, progress[:0]), ok),
                       (([p], [g], m, v, progress.float()), ok), (([p], [g], m, new_state([p], 8)[1], progress), ok),
                       (([p], [g], m, v, progress), dict(lr=-1.0)), (([p], [g], m, v, progress), dict(lr=float("nan"))),
                       (([p], [g], m, v, progress), dict(lr=1e-3, betas=(1.0, 0.9))),
                       (([p], [g], m, v, progress), dict(lr=1e-3, clip=p[:2].double())),
                       (([p], [g], m, v, progress), dict(lr=p[:2]))):
        with pytest.raises(ValueError):
            adamw_step(*args, **more)
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            gradient_norm([g], bad)
    with pytest.raises(ValueError):
        gradient_norm([None])
    with pytest.raises(ValueError):
        new_state([p], 16)
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(p)], moment_bits=4)
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(p)], max_grad_norm=0.0)
    assert torch.equal(moment_values(*new_state([p], 8)[:2])[0], torch.zeros(512, device=gpu, dtype=torch.bfloat16))
    # non-contiguous gradients are read as they are
    a, b = torch.zeros(20, 15, device=gpu), torch.zeros(20, 15, device=gpu)
    gt = torch.randn(15, 20, device=gpu).t()
    sa, sb = new_state([a]), new_state([b])
    adamw_step([a], [gt], *sa, **ok)
    adamw_step([b], [gt.contiguous()], *sb, **ok)
    assert torch.equal(a, b)
