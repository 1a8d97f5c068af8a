"""The model with layer norms in its radial networks and a table of pairs of species (``radial_norm``,
``edge_species``), trained with Muon and AdamW together: the path that runs all of them.

The kernels against the same model with plain torch formulas in their place (the suite's tolerances: energies
1e-5, forces and training gradients 1e-4), forces against differences of the energy, smoothness at the cutoff,
covariance under rotation, radial streaming, captured against eager training, states, and a frozen evaluation after a
step (its caches of derived weights must see the update)."""
import copy

import pytest
import torch

from conftest import RTOL_FORCE, assert_rel

pytestmark = pytest.mark.gpu

ZS = (1, 6, 8)


def _setup(gpu, *, channels=32, atoms=40, interactions=2, seed=3, edge_species=True, block_norm=False, **more):
    from mace_hip import create_model, radius_graph, sequential_insertion
    model = create_model(channels=channels, lmax=2, num_interactions=interactions, correlation=2, atomic_numbers=ZS,
                         cutoff=4.0, avg_num_neighbors=12.0, device=gpu, seed=seed, radial_norm=True,
                         edge_species=edge_species, block_norm=block_norm, **more)
    gen = torch.Generator(device=gpu).manual_seed(seed)
    with torch.no_grad():          # off the identity: every norm's weight and bias matters
        for interaction in model.interactions:
            for module in list(interaction.fc)[1:-1:2]:
                for p in module.parameters():
                    p.add_(torch.randn(p.shape, device=gpu, generator=gen) * 0.2)
    st = sequential_insertion(atoms, 0.05, min_separation=1.2, num_species=len(ZS), seed=seed)
    src, dst, shifts = radius_graph(st.positions, st.cell, 4.0)
    graph = dict(positions=st.positions.to(gpu), atomic_numbers=torch.tensor(ZS)[st.species].to(gpu),
                 batch=torch.zeros(atoms, dtype=torch.int64, device=gpu), edge_src=src.to(gpu),
                 edge_dst=dst.to(gpu), edge_shifts=shifts.to(gpu), cell=st.cell[None].to(gpu))
    return model, graph


def _plain(monkeypatch):
    from mace_hip import model as module

    def norm(x, weight, bias, *, eps=1e-5, activation=None):
        xc = x - x.mean(1, keepdim=True)
        z = weight * xc / (xc.square().mean(1, keepdim=True) + eps).sqrt() + bias
        return z * torch.sigmoid(z)

    monkeypatch.setattr(module, "layer_norm", norm)
    monkeypatch.setattr(module, "embedding", lambda tokens, table: table[tokens])


def _both(model):
    from ictc_o3.optim import AdamW, Muon, Together
    from mace_hip import split_parameters
    matrices, others = split_parameters(model)
    return Together(Muon(matrices, lr=0.02, weight_decay=0.01), AdamW(others, lr=1e-3, max_grad_norm=10.0))


@pytest.mark.parametrize("edge_species,block_norm", [(True, False), (False, True)])
def test_model_matches_plain_formulas(gpu, monkeypatch, edge_species, block_norm):
    from mace_hip import energy_and_forces, force_loss
    from mace_hip.runtime import backward_to_parameters
    model, graph = _setup(gpu, edge_species=edge_species, block_norm=block_norm)
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


def test_forces_are_the_energys_slope(gpu):
    """Along a random direction; float32 energies of order 10 and a step of 1e-2: 1e-6 * 10 / 2e-2 of rounding."""
    from mace_hip import energy_and_forces
    model, graph = _setup(gpu)
    model.requires_grad_(False)
    v = torch.randn(40, 3, generator=torch.Generator().manual_seed(1)).to(gpu)
    v /= v.norm()
    slope = -(energy_and_forces(model, **graph)["forces"] * v).sum().item()
    ends = [energy_and_forces(model, **{**graph, "positions": graph["positions"] + h * v})["energy"].double().sum().item()
            for h in (1e-2, -1e-2)]
    assert slope == pytest.approx((ends[0] - ends[1]) / 2e-2, rel=5e-3, abs=5e-3)


def test_edges_fade_out_at_the_cutoff(gpu):
    """Two atoms at nearly the cutoff's distance have the energies of single ones, and no force."""
    from mace_hip import energy_and_forces
    model, _ = _setup(gpu)
    model.requires_grad_(False)

    def pair(r, edges=True):
        pos = torch.tensor([[0.0, 0.0, 0.0], [0.0, 0.0, r]], device=gpu)
        src, dst = torch.tensor([[0, 1], [1, 0]] if edges else [[], []], dtype=torch.int64, device=gpu)
        return energy_and_forces(model, pos, torch.tensor([1, 6], device=gpu), torch.zeros(2, dtype=torch.int64, device=gpu),
                                 src, dst, torch.zeros(len(src), 3, device=gpu), 50.0 * torch.eye(3, device=gpu)[None])

    alone, near, close = pair(4.0, False), pair(3.9999), pair(2.0)
    assert_rel(near["energy"], alone["energy"], rtol=1e-6)
    assert near["forces"].abs().max() <= 1e-4 * close["forces"].abs().max()
    assert (close["energy"] - alone["energy"]).abs() > 1e-3


def test_rotation(gpu):
    from mace_hip import energy_and_forces
    model, graph = _setup(gpu)
    gen = torch.Generator().manual_seed(0)
    q = torch.linalg.qr(torch.randn(3, 3, generator=gen, dtype=torch.float64))[0].float().to(gpu)
    a = energy_and_forces(model, **graph)
    b = energy_and_forces(model, **{**graph, "positions": graph["positions"] @ q.T, "cell": graph["cell"] @ q.T})
    assert_rel(b["energy"], a["energy"], what="energy")
    assert_rel(b["forces"], a["forces"] @ q.T, rtol=RTOL_FORCE, what="forces")


def test_streaming_and_one_stream(gpu):
    from mace_hip import energy_and_forces
    model, graph = _setup(gpu)
    want = energy_and_forces(model, **graph)
    model.overlap_radial = False
    one = energy_and_forces(model, **graph)
    model.set_message_streaming(100)
    streamed = energy_and_forces(model, **graph)
    for out in (one, streamed):
        assert_rel(out["energy"], want["energy"])
        assert_rel(out["forces"], want["forces"], rtol=RTOL_FORCE)


def test_split_parameters(gpu):
    from mace_hip import split_parameters
    model, _ = _setup(gpu, block_norm=True)
    names = {id(p): n for n, p in model.named_parameters()}
    matrices, others = ([names[id(p)] for p in ps] for ps in split_parameters(model))
    assert len(matrices) + len(others) == sum(p.requires_grad for p in model.parameters())
    for part in ("interactions.0.fc.0.weight", "interactions.1.linear_up.weights.2", "products.0.linear.weights.0",
                 "interactions.0.self_connection.weight", "block_gates.1.weight", "last_readout.0.weight",
                 "interactions.1.message_linear.weights.1"):
        assert part in matrices, part
    for part in ("node_embedding.weight", "interactions.0.fc.1.weight", "interactions.1.edge_embedding",
                 "block_post_norms.0", "layer_readouts.0.weight", "last_readout.2.weight", "input_norm"):
        assert part in others, part
    assert all("symmetric_contractions" in n or n in others for n in others)


def test_captured_training_matches_eager(gpu):
    from mace_hip import CapturedTrainingStep, energy_and_forces, training_step
    first, graph = _setup(gpu)
    second = copy.deepcopy(first)
    eager, captured = _both(first), _both(second)
    for _ in range(2):
        training_step(first, eager, graph)
        training_step(second, captured, graph)
    step = CapturedTrainingStep(second, captured, graph, warmup=2)
    for _ in range(2):
        training_step(first, eager, graph)
    gen = torch.Generator(device=gpu).manual_seed(9)
    for k in range(3):
        pos = graph["positions"] + 0.02 * torch.randn(40, 3, device=gpu, generator=gen)
        want = training_step(first, eager, {**graph, "positions": pos})
        got = step(pos)
        torch.cuda.synchronize()
        assert_rel(got, want, rtol=1e-4, what=f"loss {k}")
    for (name, a), b in zip(first.named_parameters(), second.parameters()):
        assert_rel(b, a, rtol=1e-3, what=name)
    # a frozen evaluation goes by the weights as they are now
    frozen = copy.deepcopy(second).requires_grad_(False)
    assert_rel(energy_and_forces(second.requires_grad_(False), **graph)["energy"], energy_and_forces(frozen, **graph)["energy"])


def test_runs_agree_in_bits(gpu):
    from mace_hip import training_step
    results = []
    for _ in range(2):
        model, graph = _setup(gpu)
        optimizer = _both(model)
        for _ in range(3):
            training_step(model, optimizer, graph)
        results.append([p.detach().clone() for p in model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_states(gpu):
    """A state that is loaded goes on as the optimizer it came from; buffers of a captured step stay in place."""
    from ictc_o3.optim import Muon
    from mace_hip import split_parameters, training_step
    model, graph = _setup(gpu)
    optimizer = _both(model)
    for _ in range(2):
        training_step(model, optimizer, graph)
    twin = copy.deepcopy(model)
    other = _both(twin)
    other.load_state_dict(copy.deepcopy(optimizer.state_dict()))
    late = copy.deepcopy(model)
    third = _both(late)
    training_step(late, third, graph)
    with torch.no_grad():
        for p, q in zip(late.parameters(), model.parameters()):
            p.copy_(q)
    buffers = {p: s["momentum_buffer"] for p, s in third.optimizers[0].state.items()}
    third.load_state_dict(copy.deepcopy(optimizer.state_dict()))
    assert all(third.optimizers[0].state[p]["momentum_buffer"] is b for p, b in buffers.items())
    for m, o in ((model, optimizer), (twin, other), (late, third)):
        training_step(m, o, graph)
    for a, b, c in zip(model.parameters(), twin.parameters(), late.parameters()):
        assert torch.equal(a, b) and torch.equal(a, c)
    muon = Muon(split_parameters(model)[0][:2], lr=0.1)
    with pytest.raises(ValueError):
        muon.load_state_dict(optimizer.optimizers[0].state_dict())


def test_first_muon_step_cannot_be_captured(gpu):
    from ictc_o3.optim import Muon
    p = torch.nn.Parameter(torch.randn(16, 16, device=gpu))
    p.grad = torch.randn(16, 16, device=gpu)
    optimizer = Muon([p], lr=torch.tensor(0.1, device=gpu))
    with pytest.raises(RuntimeError), torch.cuda.graph(torch.cuda.CUDAGraph()):
        optimizer.step()
    assert not optimizer.state
    before = p.detach().clone()
    optimizer.step()
    assert not torch.equal(p, before) and optimizer.param_groups[0]["capturable"]


def test_option_refusals(gpu):
    from ictc_o3.optim import AdamW, Together
    from mace_hip import create_model
    with pytest.raises(ValueError):
        create_model(channels=8, lmax=1, device=gpu, edge_species=True)
    with pytest.raises(ValueError):
        Together()
    p = torch.nn.Parameter(torch.zeros(4, 4, device=gpu))
    with pytest.raises(ValueError):
        Together(AdamW([p]), AdamW([p]))
