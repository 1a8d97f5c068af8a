"""The optimizer's own bookkeeping, without a GPU: what a loaded state, a copy and a capture do to it."""
import copy
import pickle

import pytest
import torch

from ictc_o3.optim import AdamW


def _params(count=2):
    return [torch.nn.Parameter(torch.full((3,), float(k))) for k in range(count)]


def test_a_loaded_state_keeps_the_rate_tensors():
    """A captured step reads the rate at its tensor's address: the loaded value goes there."""
    own, shared = torch.tensor([1e-2]), torch.tensor(1e-3)
    make = lambda a, b: AdamW([{"params": p[:1], "lr": a}, {"params": p[1:]}], lr=b)      # noqa: E731
    p = _params(3)
    optimizer = make(own, shared)
    other = make(torch.tensor(0.5), torch.tensor(0.25))
    optimizer.load_state_dict(other.state_dict())
    assert optimizer.param_groups[0]["lr"] is own and optimizer.param_groups[1]["lr"] is shared
    assert own.item() == 0.5 and shared.item() == 0.25
    optimizer.load_state_dict(make(0.125, 2.0).state_dict())        # numbers, into the tensors
    assert optimizer.param_groups[0]["lr"] is own and own.item() == 0.125 and shared.item() == 2.0
    assert other.param_groups[0]["lr"].item() == 0.5                # the saved state's own is not shared


def test_a_loaded_rate_tensor_goes_beside_the_parameters():
    """From a state on another device, into a group whose rate was a number."""
    p = _params(1)
    saved = AdamW(p, lr=torch.tensor(0.5)).state_dict()
    optimizer = AdamW([torch.nn.Parameter(torch.empty(3, device="meta"))], lr=1e-3)
    optimizer.load_state_dict(saved)
    assert optimizer.param_groups[0]["lr"].device.type == "meta"


def test_groups_that_share_a_rate_tensor_take_one_value():
    p, rate = _params(2), torch.tensor(1e-3)
    optimizer = AdamW([{"params": p[:1]}, {"params": p[1:]}], lr=rate, weight_decay=0.25)
    same = AdamW([{"params": p[:1]}, {"params": p[1:]}], lr=0.5)
    optimizer.load_state_dict(same.state_dict())
    assert all(g["lr"] is rate for g in optimizer.param_groups) and rate.item() == 0.5
    two = AdamW([{"params": p[:1], "lr": 1.0}, {"params": p[1:], "lr": 2.0}], weight_decay=0.125)
    before = optimizer.param_groups[0]["weight_decay"]
    with pytest.raises(ValueError, match="share"):
        optimizer.load_state_dict(two.state_dict())
    assert rate.item() == 0.5 and optimizer.param_groups[0]["weight_decay"] == before     # nothing was taken over


def test_a_first_step_is_refused_in_a_capture(monkeypatch):
    """The moments' zeros would be part of the graph, and every replay a first step."""
    p = _params(1)
    p[0].grad = torch.ones(3)
    for clipped in (None, 1.0):
        optimizer = AdamW(p, max_grad_norm=clipped)
        monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="first step"):
            optimizer.step()
        assert optimizer.moments(p[0]) is None
    p[0].grad = None
    optimizer.step()                                     # nothing to do


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_copies_keep_everything(copied):
    p = _params()
    optimizer = AdamW([{"params": p[:1], "lr": 0.5}, {"params": p[1:]}], moment_bits=8, max_grad_norm=3.0, seed=11)
    codes = lambda k: (torch.full((256,), k, dtype=torch.uint8), torch.ones(1, dtype=torch.uint8))       # noqa: E731
    optimizer._moments[1] = (codes(3), codes(5), torch.full((1, 3), 7.0, dtype=torch.float64))
    q, other = copied((p, optimizer))
    assert (other.moment_bits, other.max_grad_norm, other.seed) == (8, 3.0, 11) and other.grad_norm is None
    assert other.param_groups[0]["lr"] == 0.5 and other.param_groups[1]["params"][0] is q[1]
    assert other._moments[0] is None and other._moments[1][0][0].eq(3).all()
    other._moments[1][2].zero_()
    assert optimizer._moments[1][2].eq(7.0).all()                    # tensors of its own
    other.step()                                                     # (no gradients)
    state = other.state_dict()
    assert state["seed"] == 11 and state["moments"][0] is None


def test_parameters_that_are_not_contiguous_are_refused_when_they_are_given():
    p = _params(1)
    bad = torch.nn.Parameter(torch.zeros(4, 3).t())
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([*p, bad])
    optimizer = AdamW(p)
    with pytest.raises(ValueError, match="contiguous"):
        optimizer.add_param_group({"params": [bad]})
    assert len(optimizer.param_groups) == len(optimizer._moments) == 1
    optimizer.add_param_group({"params": torch.nn.Parameter(torch.zeros(2, 2))})       # a tensor by itself
    assert len(optimizer.param_groups) == len(optimizer._moments) == 2


def test_a_parameter_is_in_a_group_once():
    """One launch updates all of a group's tensors side by side: twice the same one would race with itself."""
    p = _params()
    with pytest.raises(ValueError, match="once"):
        AdamW([p[0], p[1], p[0]])
