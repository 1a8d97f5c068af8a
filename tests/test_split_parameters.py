"""Which of a model's parameters are matrices for Muon, without a GPU: every trained parameter is in one of the two
lists, and tables, contraction weights, norms, path weights and maps of one output are in the other one."""
import pytest


@pytest.mark.parametrize("block_norm,radial_norm,edge_species", [(False, False, False), (True, True, True), (False, True, False)])
def test_every_parameter_is_in_one_list(block_norm, radial_norm, edge_species):
    from mace_hip import create_model, split_parameters
    model = create_model(channels=16, lmax=2, num_interactions=3, correlation=2, device="cpu", seed=0, block_norm=block_norm,
                         radial_norm=radial_norm, edge_species=edge_species)
    model.interactions[1].linear_up.weights[0].requires_grad_(False)
    names = {id(p): n for n, p in model.named_parameters() if p.requires_grad}
    matrices, others = split_parameters(model)
    listed = [names[id(p)] for p in matrices + others]
    assert sorted(listed) == sorted(names.values()) and len(set(listed)) == len(listed)
    for p in matrices:
        name = names[id(p)]
        assert p.dim() >= 2 and min(p.shape[-2:]) > 1 and p.is_contiguous(), name
        assert not any(part in name for part in ("symmetric_contractions", "norm", "embedding", "tp.weight", "readouts")), name
    for p in others:
        name = names[id(p)]
        assert not any(part in name for part in ("linear_up", "message_linear", "self_connection", "products.0.linear", "fc.0.",
                                                 "fc.2.", "fc.4.", "fc.6.")) or p.dim() < 2 or min(p.shape[-2:]) == 1, name
    assert len(matrices) > 20
