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
