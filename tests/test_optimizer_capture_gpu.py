"""The optimizer's step in a captured graph: what replays do after the optimizer's state has been changed."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = (300, 7, 1025)


def _optimizer(gpu, bits, lr=1e-2, seed=0):
    from ictc_o3.optim import AdamW
    gen = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(n, generator=gen).to(gpu)) for n in SIZES]
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen).to(gpu)
    return params, AdamW(params, lr=torch.tensor(lr, device=gpu), moment_bits=bits, max_grad_norm=1.0)


def _captured(optimizer):
    """The step as a graph (after one step outside of it, which makes the moments)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        optimizer.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optimizer.step()
    return graph


@pytest.mark.parametrize("where", ["cuda", "cpu"])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_goes_on_from_a_loaded_state(gpu, bits, where):
    """Moments, steps and the learning rate are the loaded ones, and a later change of the rate is seen."""
    params, optimizer = _optimizer(gpu, bits)
    graph = _captured(optimizer)
    graph.replay()
    torch.cuda.synchronize()
    others, other = _optimizer(gpu, bits, lr=0.25, seed=1)
    for _ in range(2):
        other.step()
    saved = other.state_dict()
    if where == "cpu":
        saved["moments"] = [tuple(tuple(t.cpu() for t in part) if isinstance(part, tuple) else part.cpu()
                                  for part in state) for state in saved["moments"]]
        saved["param_groups"] = [{**g, "lr": g["lr"].cpu()} for g in saved["param_groups"]]
    optimizer.load_state_dict(saved)
    with torch.no_grad():
        for a, b in zip(params, others):
            a.copy_(b)
            a.grad.copy_(b.grad)
    for step, rate in enumerate((None, 0.5, 0.125)):
        if rate is not None:
            optimizer.param_groups[0]["lr"].fill_(rate)
            other.param_groups[0]["lr"].fill_(rate)
        graph.replay()
        torch.cuda.synchronize()
        other.step()
        torch.cuda.synchronize()
        for a, b in zip(params, others):
            assert torch.equal(a, b), step
    assert float(optimizer.moments(params[2])[2]) == 5.0


@pytest.mark.parametrize("bits", [32, 8])
def test_a_first_step_cannot_be_captured(gpu, bits):
    """Neither a new optimizer's nor that of a group without a gradient until now; the refusal changes nothing."""
    params, optimizer = _optimizer(gpu, bits)
    before = [p.detach().clone() for p in params]
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            optimizer.step()
    late = torch.nn.Parameter(torch.ones(40, device=gpu))
    optimizer.add_param_group({"params": [late]})
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(params, before)) and optimizer.moments(params[0]) is None
    graph = _captured(optimizer)                 # the second group has no gradient: not part of it
    late.grad = torch.ones_like(late)
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            optimizer.step()
    late.grad = None
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    assert float(optimizer.moments(params[1])[2]) == 4.0


def test_a_training_step_needs_a_step_before_its_capture(gpu):
    from ictc_o3.optim import AdamW
    from mace_hip import CapturedTrainingStep, training_step
    from test_mace_gpu import _setup
    model, graph, _, _ = _setup(gpu, atoms=32)
    species = model.species_index(graph["atomic_numbers"])
    optimizer = AdamW(model.parameters(), lr=1e-3)
    # the model's own first call (its checks read from the device)
    training_step(model, torch.optim.SGD(model.parameters(), lr=0.0), dict(graph), species=species)
    with pytest.raises(RuntimeError, match="first step"):
        CapturedTrainingStep(model, optimizer, graph, species=species, warmup=0)
    model.zero_grad(set_to_none=True)
    training_step(model, optimizer, dict(graph))
    first = next(p for p in model.parameters() if p.requires_grad)
    assert float(optimizer.moments(first)[2]) == 1.0
    captured = CapturedTrainingStep(model, optimizer, graph, warmup=1)
    for _ in range(2):
        captured(graph["positions"])
        torch.cuda.synchronize(gpu)
    assert float(optimizer.moments(first)[2]) == 4.0


@pytest.mark.parametrize("bits", [32, 8])
def test_a_copy_goes_on_by_itself(gpu, bits):
    import copy
    params, optimizer = _optimizer(gpu, bits)
    optimizer.step()
    others, other = copy.deepcopy((params, optimizer))
    for a, b in zip(params, others):
        b.grad = a.grad.clone()
    other.step()
    optimizer.step()
    assert all(torch.equal(a, b) for a, b in zip(params, others))
    assert torch.equal(optimizer.grad_norm, other.grad_norm)
    other.step()
    assert float(optimizer.moments(params[0])[2]) == 2.0 and float(other.moments(others[0])[2]) == 3.0


@pytest.mark.parametrize("fused", [False, True])
def test_a_frozen_evaluation_sees_replayed_steps(gpu, fused):
    """What a frozen model derives from its weights once and keeps (folded gate weights, contraction tables) goes
    by the weights' versions: replays have to raise them as eager steps do."""
    import copy
    from conftest import RTOL_FORCE, assert_rel
    from ictc_o3.optim import AdamW
    from mace_hip import CapturedTrainingStep, energy_and_forces
    from test_mace_gpu import _setup
    model, graph, _, _ = _setup(gpu, atoms=48)
    trained = [p for p in model.parameters() if p.requires_grad]
    optimizer = torch.optim.AdamW(trained, lr=0.02, capturable=True, fused=True) if fused else AdamW(trained, lr=0.02)
    captured = CapturedTrainingStep(model, optimizer, graph, warmup=1)

    def frozen(m):
        for p in m.parameters():
            p.requires_grad_(False)
        return energy_and_forces(m, **graph)

    first = frozen(model)
    for _ in range(3):
        for p in trained:
            p.requires_grad_(True)
        captured(graph["positions"])
        torch.cuda.synchronize(gpu)
        got, want = frozen(model), frozen(copy.deepcopy(model))      # (a copy derives its own)
        assert_rel(got["energy"], want["energy"], what="energy")
        assert_rel(got["forces"], want["forces"], rtol=RTOL_FORCE, what="forces")
    assert not torch.allclose(got["energy"], first["energy"], rtol=1e-3)


@pytest.mark.parametrize("limit", [1e-40, 1e-46, 1e-300])
def test_limits_below_float32_are_limits(gpu, limit):
    """Below float32's smallest number a limit was passed as zero, which means none."""
    from ictc_o3 import gradient_norm
    norm, coefficient = gradient_norm([torch.full((30,), 3.0, device=gpu)], limit).tolist()
    assert abs(norm - 270.0 ** 0.5) <= 2e-6 * norm and 0.0 <= coefficient <= 2e-41
