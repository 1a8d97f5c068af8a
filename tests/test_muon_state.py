"""States of ``ictc_o3.optim.Muon`` without a GPU: torch's own Muon and this one take each other's, and what is no Muon's
state is refused before anything changes."""
import copy

import pytest
import torch


def _params():
    g = torch.Generator().manual_seed(0)
    return [torch.nn.Parameter(torch.randn(*s, generator=g)) for s in ((4, 6), (5, 5), (3, 2))]


def _stepped():
    params = _params()
    theirs = torch.optim.Muon(params, lr=0.03, momentum=0.9, weight_decay=0.02, ns_steps=6)
    for p in params[:2]:
        p.grad = torch.ones_like(p)
    theirs.step()
    return theirs


def test_torch_states_are_taken():
    from ictc_o3.optim import Muon
    theirs, params = _stepped(), _params()
    own = Muon(params, lr=0.5)
    own.load_state_dict(theirs.state_dict())
    group = own.param_groups[0]
    assert group["capturable"] and group["adjust_lr_fn"] is None
    assert (group["lr"], group["momentum"], group["weight_decay"], group["ns_steps"]) == (0.03, 0.9, 0.02, 6)
    for p, q in zip(params, theirs.param_groups[0]["params"]):
        assert (p in own.state) == (q in theirs.state)
        if p in own.state:
            a, b = own.state[p]["momentum_buffer"], theirs.state[q]["momentum_buffer"]
            assert torch.equal(a, b) and a is not b
    back = torch.optim.Muon(_params())
    back.load_state_dict(copy.deepcopy(own.state_dict()))
    assert back.param_groups[0]["lr"] == 0.03 and len(back.state) == 2
    assert Muon(_params(), adjust_lr_fn=None).param_groups[0]["adjust_lr_fn"] is None


def test_other_states_are_refused():
    from ictc_o3.optim import AdamW, Muon
    params = _params()
    own = Muon(params, lr=0.5)
    own.load_state_dict(_stepped().state_dict())
    before = copy.deepcopy(own.state_dict())
    adam = torch.optim.AdamW(_params())
    for p in adam.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    adam.step()
    half = copy.deepcopy(before)
    half["state"][1] = {"step": 1}
    for state in (adam.state_dict(), AdamW(_params()).state_dict(), torch.optim.SGD(_params(), lr=0.1).state_dict(), half):
        with pytest.raises(ValueError, match="not that of a Muon"):
            own.load_state_dict(state)
    after = own.state_dict()
    assert after["param_groups"] == before["param_groups"]
    assert all(torch.equal(after["state"][k]["momentum_buffer"], s["momentum_buffer"]) for k, s in before["state"].items())
