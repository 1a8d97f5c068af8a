"""The composed gradient formula of the block norms (third derivatives, cotangents of weight gradients) on the CPU:
float32 operands against the same formula on float64 copies of them.

Its result differs from the exact one by the rounding of float32 results only (1 u = 6e-8 of an entry) where statistics
and projections are in 64 bits; the suite's 1e-5 of the largest entry leaves no room for a cotangent's part along
the row, which cancels down to eps / (q + eps) of it for a row with one large entry."""
import pytest
import torch

from conftest import assert_rel


def _operands(c, lmax, rows, one_large):
    g = torch.Generator().manual_seed(10 * c + lmax)
    width, places = c * (lmax + 1) ** 2, c * (lmax + 1)
    draw = lambda *s: torch.randn(*s, generator=g)       # noqa: E731
    t = [draw(rows, width), 2 * draw(rows, width), draw(rows, places), 1 + 0.2 * draw(places), 1 + 0.2 * draw(places),
         draw(rows, width), draw(rows, width)]
    if one_large:
        t[0][:, -1] = t[1][:, -1] = 300.0
    return t, [draw(rows, width), draw(rows, width), draw(rows, places), draw(places), draw(places)]


@pytest.mark.parametrize("block", [True, False])
@pytest.mark.parametrize("c,lmax,rows,one_large", [(1, 0, 7, False), (1, 0, 7, True), (5, 1, 6, True),
                                                   (6, 2, 11, False)])
def test_formula_in_single_precision(c, lmax, rows, one_large, block):
    from ictc_o3 import _lib
    from ictc_o3.backends.hip.norms import gradient_formula
    values, cots = _operands(c, lmax, rows, one_large)
    results = []
    for dtype in (torch.float32, torch.float64):
        t = [v.to(dtype).requires_grad_() for v in values]
        if not block:
            t[1] = t[2] = t[3] = t[5] = None
        first = gradient_formula(_lib.NormDesc(c, lmax, lmax, 0.7, 1e-5), *t)
        assert all(f is None or f.dtype == dtype for f in first)
        heads = [(f, k.to(dtype)) for f, k in zip(first, cots) if f is not None]
        second = torch.autograd.grad([f for f, _ in heads], [v for v in t if v is not None], [k for _, k in heads],
                                     create_graph=True, allow_unused=True)
        third = torch.autograd.grad(sum(s.square().sum() for s in second if s is not None),
                                    [v for v in t if v is not None], allow_unused=True)
        results.append([*first, *second, *third])
    for k, (got, want) in enumerate(zip(*results)):
        assert (got is None) == (want is None)
        if want is not None:
            assert_rel(got, want, what=f"result {k}")
