"""Stacks of one, three and four interactions: a frozen model (whose last two readouts are one kernel) gives the
energies and forces that the trainable one gives."""
import copy

import pytest
import torch

from conftest import RTOL_FORCE, assert_rel

pytestmark = pytest.mark.gpu

ZS = (1, 6, 8)


@pytest.mark.parametrize("interactions", [1, 3, 4])
def test_frozen_and_trainable_energies_agree(gpu, interactions):
    from mace_hip import create_model, energy_and_forces, radius_graph, sequential_insertion
    model = create_model(channels=16, lmax=1, num_interactions=interactions, correlation=2, atomic_numbers=ZS, cutoff=4.0,
                         avg_num_neighbors=12.0, device=gpu, seed=1)
    st = sequential_insertion(30, 0.05, min_separation=1.2, num_species=len(ZS), seed=1)
    src, dst, shifts = radius_graph(st.positions, st.cell, 4.0)
    graph = dict(positions=st.positions.to(gpu), atomic_numbers=torch.tensor(ZS)[st.species].to(gpu),
                 batch=torch.zeros(30, dtype=torch.int64, device=gpu), edge_src=src.to(gpu), edge_dst=dst.to(gpu),
                 edge_shifts=shifts.to(gpu), cell=st.cell[None].to(gpu))
    want = energy_and_forces(model, **graph)
    got = energy_and_forces(copy.deepcopy(model).requires_grad_(False), **graph)
    assert got["atomic_energy"].shape == want["atomic_energy"].shape == (30,)
    assert_rel(got["atomic_energy"], want["atomic_energy"], what="atomic energies")
    assert_rel(got["forces"], want["forces"], rtol=RTOL_FORCE, what="forces")
