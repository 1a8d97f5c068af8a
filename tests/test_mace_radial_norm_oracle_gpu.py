"""The model with layer norms in its radial networks and a table of pairs of species against the float64 oracle on the
CPU, which holds none of this repository's kernels: the gates alone (where the envelope, the pairs' rows and the last
weight's factor stand), energies, forces and the force loss's gradients (the suite's tolerances)."""
import pytest
import torch

from conftest import RTOL_FORCE, assert_rel
from oracle.mace import MaceOracle, bessel_features
from test_mace_radial_norm_gpu import ZS, _setup

pytestmark = pytest.mark.gpu


def _both(gpu, edge_species, **more):
    model, graph = _setup(gpu, edge_species=edge_species, **more)
    state = [*model.named_parameters(), *model.named_buffers()]
    oracle = MaceOracle({k: v.detach().double().cpu() for k, v in state}, channels=32, lmax=2,
                        num_interactions=len(model.interactions), correlation=2, num_elements=len(ZS), cutoff=4.0,
                        avg_num_neighbors=12.0)
    species = model.species_index(graph["atomic_numbers"]).cpu()
    cpu = dict(pos=graph["positions"].double().cpu(), species=species, src=graph["edge_src"].cpu(),
               dst=graph["edge_dst"].cpu(), shifts=graph["edge_shifts"].double().cpu(), cell=graph["cell"].double().cpu(),
               batch=graph["batch"].cpu())
    return model, graph, oracle, cpu


@pytest.mark.parametrize("edge_species", [True, False])
def test_gates(gpu, edge_species):
    """Of edges of all lengths up to the cutoff and beyond it, and of each pair of species; both forms that the
    interaction gives its radial network in."""
    from mace_hip.model import EdgeExtras
    from mace_hip.radial import cutoff_envelope
    model, _, oracle, _ = _both(gpu, edge_species)
    g = torch.Generator().manual_seed(0)
    r = torch.linspace(0.3, 4.4, 900, dtype=torch.float64)
    pairs = torch.randint(len(ZS) ** 2, (900,), generator=g)
    feats = bessel_features(r, 4.0, 8, 5)
    vec = torch.zeros(900, 3, dtype=torch.float64)
    vec[:, 2] = r
    extras = EdgeExtras(cutoff_envelope(vec, 4.0, 5).float().to(gpu), pairs.to(gpu) if edge_species else None)
    for t, interaction in enumerate(model.interactions):
        want = oracle.radial_gates(f"interactions.{t}", feats, r, pairs)
        assert not want[r > 4.0].any() and want[r < 3.0].abs().max() > 0.1
        hidden, weight = interaction.radial_hidden(feats.float().to(gpu), extras)
        for got in (interaction.radial_mlp(feats.float().to(gpu), extras), hidden @ weight.t()):
            assert_rel(got, want, what="gates")
        weighted = interaction.message_gates(feats.float().to(gpu), extras)
        assert_rel(weighted, want * oracle.p[f"interactions.{t}.tp.weight"].reshape(1, -1), what="weighted gates")


@pytest.mark.parametrize("edge_species,interactions", [(True, 2), (False, 2), (True, 3)])
def test_energies_forces_and_gradients(gpu, edge_species, interactions):
    from mace_hip import energy_and_forces, force_loss
    model, graph, oracle, cpu = _both(gpu, edge_species, interactions=interactions)
    pred = energy_and_forces(model, **graph, training=True)
    loss = force_loss(pred, 40)
    loss.backward()
    names = [n for n, p in model.named_parameters() if p.requires_grad]
    for n in names:
        oracle.p[n].requires_grad_(True)
    e, f, atomic = oracle.energy_and_forces(**cpu, create_graph=True)
    assert_rel(pred["atomic_energy"], atomic, what="atomic energies")
    assert_rel(pred["energy"], e, what="energy")
    assert_rel(pred["forces"], f, rtol=RTOL_FORCE, what="forces")
    want = torch.autograd.grad((e / 40).square().mean() + f.square().mean(), [oracle.p[n] for n in names])
    params = dict(model.named_parameters())
    for n, g in zip(names, want):
        assert_rel(params[n].grad, g, rtol=RTOL_FORCE, what=f"d loss / d {n}")
