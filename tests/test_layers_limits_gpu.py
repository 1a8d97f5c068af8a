"""Layer norm, embedding and orthogonalised updates at the ends of what they take: stacks of matrices that are split,
tables on both sides of the rule by which their tokens are sorted, matrices of float32's largest and smallest numbers."""
import pytest
import torch

from test_embedding_gpu import _case, _check_gradient
from test_muon_gpu import _check, _exact

pytestmark = pytest.mark.gpu


def _draw(shape, seed, gpu, scale=1.0):
    return scale * torch.randn(*shape, device=gpu, generator=torch.Generator(device=gpu).manual_seed(seed))


@pytest.mark.parametrize("shape,parts", [((200_000, 8, 8), 7), ((90, 300, 5000), 4)], ids=["short", "long"])
def test_stacks_in_several_groups(gpu, shape, parts):
    """A stack that takes several turns in the workspace has the bits of its parts alone, whatever lies beside it."""
    from ictc_o3.operators import orthogonalize
    u, other = _draw(shape, 1, gpu), _draw((50, 60), 2, gpu)
    got = orthogonalize([other, u, other])
    want = torch.cat([orthogonalize([p])[0] for p in u.chunk(parts)])
    assert torch.equal(got[1], want)
    assert torch.equal(got[0], got[2]) and torch.equal(got[0], orthogonalize([other])[0])


def test_steps_of_stacks_in_several_groups(gpu):
    """Parameters and momentum of every part are written once, those without a gradient not at all."""
    from ictc_o3.operators import muon_step
    shapes = [(120_000, 4, 9), (70_000, 12, 5), (3, 20, 20)]
    first = [[_draw(s, 10 * j + k, gpu, scale) for k, s in enumerate(shapes)]
             for j, scale in ((1, 0.1), (2, 0.01), (3, 0.005))]
    grads = [first[1][0], None, first[1][2]]
    second = [[t.clone() for t in ts] for ts in first]
    muon_step(first[0], grads, first[2], lr=0.1)
    for k in (0, 2):
        for p, g, m in zip(*(ts[k].chunk(5) for ts in second)):
            muon_step([p], [g], [m], lr=0.1)
    for ts, us in ((first[0], second[0]), (first[2], second[2])):
        assert all(torch.equal(t, u) for t, u in zip(ts, us))


@pytest.mark.parametrize("count,rows,width", [(40_000, 255, 64), (40_000, 255, 65), (40_000, 256, 64), (8192, 255, 256),
                                              (8193, 255, 256), (8193, 1, 256), (8193, 200, 300), (20_000, 3, 513)])
def test_few_rows_of_many_columns(gpu, count, rows, width):
    """Tolerance: test_embedding_gpu's.  Some tokens lie outside the table."""
    from ictc_o3.operators import embedding
    tokens, table, dy = _case(count, rows, width, count + rows + width)
    tokens[::13] = -1
    leaf, at, top = table.to(gpu).requires_grad_(), tokens.to(gpu), dy.to(gpu)
    first, second = (torch.autograd.grad(embedding(at, leaf, scale=0.5), leaf, top)[0] for _ in range(2))
    _check_gradient(first, tokens, dy, rows, 0.5)
    assert torch.equal(first, second)


@pytest.mark.parametrize("scale", [3.4e38, -2.5e38, 1e-42, 1e-44], ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (40, 70), (200, 300), (150, 140)], ids=str)
def test_largest_and_smallest_numbers(gpu, shape, scale):
    """Entries up to float32's last power of two, and ones that are below its normal range (then X stays far below 1).
    Tolerance: test_muon_gpu's (results are at least 3.4^5 1e-44 / eps, far above float32's smallest number)."""
    from ictc_o3.operators import orthogonalize
    u = torch.rand(*shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64) * 2 - 1
    u[0, 0] = 1.0
    u = (u * scale).float()
    assert u.isfinite().all() and u[0, 0] != 0
    got, = orthogonalize([u.to(gpu)])
    _check(got, _exact(u))


@pytest.mark.parametrize("shape", [(64, 3000), (3000, 40), (128, 2000), (300, 2000), (20, 3000)], ids=str)
def test_values_between_products_keep_both_parts(gpu, shape):
    """With coefficients (3 / 4, 0, 0) the iteration leaves X times 3 / 4 a step, through all its roundings, one by one: the
    scale's, its product, and in each step what is kept of X (2^-23, or an absolute 2^-36) and the product's: none of
    10^5 values is off by more."""
    from ictc_o3.operators import orthogonalize
    u = _draw(shape, 1, gpu)
    for steps in (1, 2, 3):
        got, = orthogonalize([u], steps=steps, coefficients=(0.75, 0.0, 0.0))
        want = u.double() / (u.double().norm() + 1e-7) * 0.75 ** steps
        bound = (2 * 2.0 ** -24 + steps * (2.0 ** -23 + 2.0 ** -24)) * 1.001 * want.abs() + steps * 2.0 ** -36
        assert bool(((got.double() - want).abs() <= bound).all()), ((got.double() - want).abs() / bound).max()


def test_zeros_with_the_smallest_eps(gpu):
    """Any positive eps is allowed: 1 / eps need not be a number."""
    from ictc_o3.operators import muon_step, orthogonalize
    shapes = [(1, 1), (5, 6), (3, 60, 70), (150, 140)]
    for got in orthogonalize([torch.zeros(*s, device=gpu) for s in shapes], eps=1e-320):
        assert not got.any()
    p, g, m = torch.ones(20, 30, device=gpu), torch.zeros(20, 30, device=gpu), torch.zeros(20, 30, device=gpu)
    muon_step([p], [g], [m], lr=0.5, weight_decay=0.5, eps=1e-320)
    assert bool((p == 0.75).all()) and not m.any()


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("width,share", [(1, 2), (8, 4), (64, 8)])
def test_many_small_sums_behind_a_large_one(gpu, rows, width, share):
    """What every group of a workgroup's lanes adds, just under half of a float32 step of the sum so far, is not lost:
    the bound of test_embedding_gpu, 64 additions in float32, whatever the number of groups."""
    from ictc_o3.operators import embedding
    dy = torch.full((512, width), 0.98 * 2.0 ** -24 / share)
    dy[:share] = 0.0
    dy[0] = 1.0
    tokens = torch.zeros(512, dtype=torch.int64)
    leaf = torch.zeros(rows, width, device=gpu, requires_grad=True)
    got, = torch.autograd.grad(embedding(tokens.to(gpu), leaf), leaf, dy.to(gpu))
    _check_gradient(got, tokens, dy, rows, 1.0)


def test_exceptions_keep_their_types(gpu, monkeypatch):
    """Memory that runs out, and what the composed formulas or a hook raise, reach the caller as what they are."""
    from ictc_o3.backends.hip import layer_norm as module
    from ictc_o3.operators import embedding, layer_norm
    with pytest.raises(torch.OutOfMemoryError):          # 800 GB
        embedding(torch.zeros(200_000, dtype=torch.int64, device=gpu), torch.zeros(2, 1 << 20, device=gpu))

    def fails(*args):
        raise KeyError("none")

    x, w = _draw((3, 8), 1, gpu).requires_grad_(), torch.ones(8, device=gpu, requires_grad=True)
    dw, = torch.autograd.grad(layer_norm(x, w), w, torch.ones(3, 8, device=gpu), create_graph=True)
    with monkeypatch.context() as patch:
        patch.setattr(module, "gradient_formula", fails)
        with pytest.raises(KeyError, match="none"):
            torch.autograd.grad(dw.sum(), x, retain_graph=True)
    assert torch.autograd.grad(dw.sum(), x)[0].shape == x.shape
    with torch.autograd.graph.saved_tensors_hooks(fails, lambda t: t), pytest.raises(KeyError, match="none"):
        layer_norm(x, w)


@pytest.mark.parametrize("radial_norm", [False, True])
def test_atoms_in_one_place(gpu, radial_norm):
    """Two atoms at the same point: energies, forces and the force loss's gradients, those to the positions among them
    (its second derivatives in the edges' lengths), are numbers."""
    from mace_hip import create_model, energy_and_forces, force_loss
    model = create_model(channels=32, lmax=2, num_interactions=2, correlation=2, cutoff=4.0, device=gpu, seed=1,
                         radial_norm=radial_norm, edge_species=radial_norm)
    pos = torch.tensor([[0.0, 0, 0], [0, 0, 0], [1.5, 0.3, 0.2], [0.1, 1.7, -0.4]], device=gpu, requires_grad=True)
    src, dst = (t.to(gpu) for t in (~torch.eye(4, dtype=torch.bool)).nonzero().unbind(1))
    out = energy_and_forces(model, pos, torch.tensor([1, 6, 8, 1], device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu),
                            src, dst, torch.zeros(12, 3, device=gpu), 50.0 * torch.eye(3, device=gpu)[None], training=True)
    force_loss(out, 4).backward()
    grads = {"positions": pos.grad, **{n: p.grad for n, p in model.named_parameters() if p.requires_grad}}
    for name, t in {**out, **grads}.items():
        assert bool(t.isfinite().all()), name


def test_steps_from_a_torch_optimizers_state(gpu):
    """A state of torch.optim.Muon (no size rule named, nothing about captures) goes on, eagerly and captured."""
    from ictc_o3.optim import Muon
    grad = _draw((20, 30), 5, gpu, 0.1)
    leaves = [torch.nn.Parameter(_draw((20, 30), 4, gpu)) for _ in range(3)]
    theirs = torch.optim.Muon([leaves[0]], lr=0.05)
    leaves[0].grad = grad.clone()
    theirs.step()
    own = [Muon([p], adjust_lr_fn=rule) for p, rule in zip(leaves[1:], (None, "original"))]
    for p, o in zip(leaves[1:], own):
        o.load_state_dict(theirs.state_dict())
        p.grad = grad.clone()
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        own[0].step()
    for _ in range(3):
        graph.replay()
        own[1].step()
        torch.cuda.synchronize()
        assert torch.equal(leaves[1], leaves[2])
    assert not torch.equal(leaves[1], _draw((20, 30), 4, gpu))


def test_bits_do_not_depend_on_company(gpu):
    """Alone (tiles of 64), and beside matrices that fill the chip (tiles of 128)."""
    from ictc_o3.operators import orthogonalize
    us = [_draw(s, k, gpu) for k, s in enumerate(((64, 300), (130, 130), (512, 200), (9, 9), (300, 257), (1024, 1024),
                                                  (3, 150, 700), (128, 129), (129, 128)))]
    many = [_draw((1024, 1024), 100, gpu)] * 10
    for a, b in zip([orthogonalize([u])[0] for u in us], orthogonalize(us + many)):
        assert torch.equal(a, b), tuple(a.shape)


def test_signs_that_are_only_noted(gpu):
    """The imaginary part of a conjugate is a view with its sign noted: taken as the numbers that it stands for, or refused
    where addresses are all that is read."""
    from ictc_o3.operators import embedding, gradient_norm, layer_norm, muon_step, orthogonalize
    z = torch.complex(torch.zeros(1, 1, device=gpu), torch.full((1, 1), 2.0, device=gpu))
    noted = torch.imag(z.conj())
    assert noted.is_neg() and noted.is_contiguous() and noted.item() == -2.0
    token, one, zero = torch.zeros(1, dtype=torch.int64, device=gpu), torch.ones(1, device=gpu), torch.zeros(1, device=gpu)
    assert embedding(token, noted).item() == -2.0
    assert layer_norm(torch.ones(1, 1, device=gpu), one, noted[0]).item() == -2.0
    leaf = torch.ones(1, 1, device=gpu, requires_grad=True)
    assert torch.autograd.grad(embedding(token, leaf), leaf, noted)[0].item() == -2.0
    bias = zero.clone().requires_grad_()
    assert torch.autograd.grad(layer_norm(leaf, one, bias), bias, noted)[0].item() == -2.0
    own = [torch.ones(1, 1, device=gpu) for _ in range(2)]
    for call in (lambda: orthogonalize([noted]), lambda: gradient_norm([noted]), lambda: muon_step([own[0]], [noted], [own[1]], lr=0.1),
                 lambda: muon_step([noted], [own[0]], [own[1]], lr=0.1)):
        with pytest.raises(ValueError):
            call()
