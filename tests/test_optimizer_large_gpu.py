"""The optimizer's launches that stream (2^24 values and more): tensors of a few blocks with tails between large ones,
some of them at odd addresses, some without a gradient, so that the groups of four blocks that a wave takes with 8-bit
moments meet tensor ends, part-filled blocks and tensors that are read value by value.  Formulas, hash and
tolerances are test_optimizer_gpu.py's."""
import pytest
import torch

import test_optimizer_gpu as small

pytestmark = pytest.mark.gpu

# (20 M values in two launches' worth of tensors, the first of which streams)
SIZES = [700, 6_000_003, 769, 1, 255, 1025, 513, 256, 1023, 0, *[1 + 97 * k % 1300 for k in range(90)], 11_000_000,
         *[1 + 131 * k % 900 for k in range(100)], 3_000_001, 40]


def _inputs(sizes, seed, gpu, offset=0):
    """test_optimizer_gpu's, every third tensor a float or three off a 16-byte boundary."""
    gen = torch.Generator(device=gpu).manual_seed(seed)
    params, grads = [], []
    for k, n in enumerate(sizes):
        off = (0, 1, 0, 0, 3, 0)[k % 6]
        draw = lambda: torch.randn(n + off, device=gpu, generator=gen)      # noqa: E731
        params.append((draw() * 0.1)[off:])
        grads.append((draw() * draw().exp() * 10.0 ** (-3 + k % 4))[off:])
    return params, grads


@pytest.fixture
def large(monkeypatch):
    assert sum(-(-n // 256) * 256 for n in SIZES[:184]) >= 1 << 24
    monkeypatch.setitem(small.SIZES, "streams", SIZES)
    monkeypatch.setattr(small, "_inputs", _inputs)


def test_steps_match_the_formula(gpu, large):
    small.test_steps_match_the_formula(gpu, "streams", 0)


def test_eight_bit_steps(gpu, large):
    small.test_eight_bit_steps(gpu, "streams", 0)


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_without_gradients(gpu, bits):
    """Left out of a launch that streams: they stay as they are, all others get the bits that they get with them."""
    from ictc_o3.backends.hip.optimizer import adamw_step, moment_values, new_state
    params, grads = _inputs(SIZES, 1, gpu)
    without = [p.clone() for p in params]
    some = [None if k in (0, 3, 4, 5, 20, 21, 22, 23, 24, 60) else g for k, g in enumerate(grads)]
    state, other = new_state(params, bits), new_state(without, bits)
    adamw_step(params, grads, *state, lr=small.LR, seed=5)
    adamw_step(without, some, *other, lr=small.LR, seed=5)
    before = _inputs(SIZES, 1, gpu)[0]
    (m, v), (m2, v2) = (s[:2] if bits == 32 else moment_values(*s[:2]) for s in (state, other))
    at = small._starts(SIZES)
    for k, n in enumerate(SIZES):
        part = slice(int(at[k]), int(at[k]) + n)
        if some[k] is None:
            assert torch.equal(without[k], before[k]) and not m2[part].any() and not v2[part].any(), k
        else:
            assert torch.equal(without[k], params[k]), k
            assert torch.equal(m2[part], m[part]) and torch.equal(v2[part], v[part]), k
    assert other[2][:, 0].tolist() == [0.0 if g is None else 1.0 for g in some]
