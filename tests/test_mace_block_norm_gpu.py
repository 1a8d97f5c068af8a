"""The model with norms, gates and a residual stream around its blocks (``block_norm``), trained with the
library's AdamW: the path that runs both together.

The kernels against the same model with plain torch formulas in their place (the suite's tolerances:
energies 1e-5, forces and training gradients 1e-4), covariance under rotation, captured against eager
training, and a frozen evaluation after a step (its caches of derived weights must see the update)."""
import copy

import pytest
import torch

from conftest import RTOL_FORCE, assert_rel
from test_norms_gpu import _block_end, _norm

pytestmark = pytest.mark.gpu

ZS = (1, 6, 8)


def _setup(gpu, *, channels=32, atoms=40, interactions=3, seed=3):
    from mace_hip import create_model, radius_graph, sequential_insertion
    model = create_model(channels=channels, lmax=2, num_interactions=interactions, correlation=2, atomic_numbers=ZS,
                         cutoff=4.0, avg_num_neighbors=12.0, device=gpu, seed=seed, block_norm=True)
    gen = torch.Generator(device=gpu).manual_seed(seed)
    with torch.no_grad():          # off the identity: every norm weight and gate matters
        for name, p in model.named_parameters():
            if "norm" in name or "gate" in name:
                p.add_(torch.randn(p.shape, device=gpu, generator=gen) * 0.2)
    st = sequential_insertion(atoms, 0.05, min_separation=1.2, num_species=len(ZS), seed=seed)
    src, dst, shifts = radius_graph(st.positions, st.cell, 4.0)
    graph = dict(positions=st.positions.to(gpu), atomic_numbers=torch.tensor(ZS)[st.species].to(gpu),
                 batch=torch.zeros(atoms, dtype=torch.int64, device=gpu), edge_src=src.to(gpu),
                 edge_dst=dst.to(gpu), edge_shifts=shifts.to(gpu), cell=st.cell[None].to(gpu))
    return model, graph


def _plain(monkeypatch):
    from mace_hip import model as module

    def norm(x, weight, *, channels, eps=1e-5):
        return _norm(x, weight.reshape(-1), channels, weight.numel() // channels - 1)

    def block_end(x, block, gate, post, pre, *, channels, residual_scale, eps=1e-5):
        return _block_end(x, block, gate, post.reshape(-1), pre.reshape(-1), channels, post.numel() // channels - 1,
                          residual_scale)

    monkeypatch.setattr(module, "equivariant_norm", norm)
    monkeypatch.setattr(module, "gated_residual_norm", block_end)


def test_model_matches_plain_formulas(gpu, monkeypatch):
    from mace_hip import energy_and_forces, force_loss
    from mace_hip.runtime import backward_to_parameters
    model, graph = _setup(gpu)
    results = []
    for plain in (False, True):
        if plain:
            _plain(monkeypatch)
        frozen = copy.deepcopy(model).requires_grad_(False)
        out = energy_and_forces(frozen, **graph)
        training = energy_and_forces(model, **graph, training=True)
        backward_to_parameters(force_loss(training, graph["positions"].shape[0]), model)
        grads = {n: p.grad for n, p in model.named_parameters() if p.requires_grad}
        model.zero_grad(set_to_none=True)
        results.append((out, training, grads))
    (out, training, grads), (out2, training2, grads2) = results
    for a in (out, training):
        assert_rel(a["energy"], out2["energy"], what="energy")
        assert_rel(a["forces"], out2["forces"], rtol=RTOL_FORCE, what="forces")
    assert all(g is not None for g in grads.values()) and len(grads) == len(grads2)
    for name, g in grads2.items():
        assert_rel(grads[name], g, rtol=RTOL_FORCE, what=name)


def test_rotation(gpu):
    from mace_hip import energy_and_forces
    model, graph = _setup(gpu)
    gen = torch.Generator().manual_seed(0)
    q = torch.linalg.qr(torch.randn(3, 3, generator=gen, dtype=torch.float64))[0].float().to(gpu)
    a = energy_and_forces(model, **graph)
    b = energy_and_forces(model, **dict(graph, positions=graph["positions"] @ q, cell=graph["cell"] @ q))
    assert_rel(b["energy"], a["energy"], what="energy")
    assert_rel(b["forces"], a["forces"] @ q, rtol=RTOL_FORCE, what="forces")


@pytest.mark.parametrize("bits", [32, 8])
def test_training_captured_and_eager(gpu, bits):
    from ictc_o3.optim import AdamW
    from mace_hip import CapturedTrainingStep, energy_and_forces, training_step
    model, graph = _setup(gpu)
    other, _ = _setup(gpu)
    make = lambda m: AdamW(m.parameters(), lr=2e-3, moment_bits=bits, max_grad_norm=10.0)    # noqa: E731
    opt, opt2 = make(model), make(other)
    losses = [training_step(model, opt, dict(graph)) for _ in range(3)]
    step = CapturedTrainingStep(other, opt2, graph, warmup=3)
    for _ in range(12):
        losses.append(training_step(model, opt, dict(graph)))
        torch.cuda.synchronize(gpu)
        replayed = step(graph["positions"]).clone()
        torch.cuda.synchronize(gpu)
        assert_rel(replayed, losses[-1], rtol=1e-3, what="loss")
    assert losses[-1] < 0.7 * losses[0]
    # a frozen evaluation right after the step: as a model built from the new parameters gives it
    model.requires_grad_(False)
    first = energy_and_forces(model, **graph)["forces"]
    model.interactions[0].fc[-1].weight.requires_grad_(True)
    loss = (energy_and_forces(model, **graph, training=True)["energy"]).square().sum()
    loss.backward()
    AdamW([model.interactions[0].fc[-1].weight], lr=0.1).step()
    model.requires_grad_(False)
    fresh = copy.deepcopy(model)
    fresh.interactions[0]._gate_weight = None
    got = energy_and_forces(model, **graph)["forces"]
    assert_rel(got, energy_and_forces(fresh, **graph)["forces"], what="forces after the step")
    assert not torch.allclose(got, first)


def test_captured_inference(gpu):
    from mace_hip import CapturedEnergyAndForces, energy_and_forces
    model, graph = _setup(gpu)
    model.requires_grad_(False)
    step = CapturedEnergyAndForces(model, **graph)
    for k in range(3):
        gen = torch.Generator(device=gpu).manual_seed(k)
        pos = graph["positions"] + 0.05 * torch.randn(graph["positions"].shape, device=gpu, generator=gen)
        eager = energy_and_forces(model, **dict(graph, positions=pos))
        torch.cuda.synchronize(gpu)
        got = step(pos)
        torch.cuda.synchronize(gpu)
        assert_rel(got["energy"], eager["energy"], what=f"replay {k} energy")
        assert_rel(got["forces"], eager["forces"], what=f"replay {k} forces")


def test_default_model_has_no_norms(gpu):
    from mace_hip import create_model
    model = create_model(channels=8, lmax=1, correlation=1, device=gpu)
    assert not any("norm" in n or "block_gates" in n for n in model.state_dict())
