"""The cutoff envelope as a function of edge vectors: values and derivatives of vectors of length zero and nearly zero,
and everywhere else those of the polynomial of the length."""
import torch


def _orders(f, vec, u):
    vec = vec.clone().requires_grad_()
    y = f(vec)
    first, = torch.autograd.grad(y.sum(), vec, create_graph=True)
    second, = torch.autograd.grad((first * u).sum(), vec, create_graph=True)
    third, = torch.autograd.grad((second * u).sum(), vec)
    return [t.detach() for t in (y, first, second, third)]


def test_vectors_of_no_length():
    """Zero, lengths whose square is below float32's range, and short ones: all derivatives are numbers."""
    from mace_hip.radial import cutoff_envelope
    vec = torch.zeros(6, 3)
    for k, size in enumerate((0.0, 1e-44, 1e-30, 1e-12, 1e-7, 3e-6)):
        vec[k, 1] = -size
    y, *rest = _orders(lambda v: cutoff_envelope(v, 4.0), vec, torch.randn(6, 3, generator=torch.Generator().manual_seed(0)))
    assert bool((y == 1.0).all())
    for t in rest:
        assert bool(t.isfinite().all()) and t.abs().max() < 1e-3


def test_other_vectors():
    """The same bits as the polynomial of the norm, also beside a vector of length zero, and nothing beyond the cutoff."""
    from mace_hip.radial import cutoff_envelope, polynomial_cutoff
    g = torch.Generator().manual_seed(1)
    vec = torch.randn(200, 3, generator=g) * 2.0
    vec[5], vec[6] = torch.tensor([4.0, 0.0, 0.0]), torch.tensor([0.0, 3e3, 0.0])
    u = torch.randn(200, 3, generator=g)
    want = _orders(lambda v: polynomial_cutoff(v.norm(dim=1), 4.0, 5), vec, u)
    got = _orders(lambda v: cutoff_envelope(v, 4.0), torch.cat([vec, torch.zeros(1, 3)]), torch.cat([u, u[:1]]))
    for a, b in zip(got, want):
        assert torch.equal(a[:200], b)
    assert want[0][5] == 0 and want[0][6] == 0
