"""The block norms' kernels where a workgroup goes on from row to row, at the widest rows, and the composed orders
behind them, against plain float64 formulas (tolerances as in test_norms_gpu.py: 1e-5 of the largest entry)."""
import pytest
import torch

from test_norms_gpu import EPS, _all_orders, _block_end, _compare, _inputs, _leaves, _norm

pytestmark = pytest.mark.gpu

NAMES = ("x", "block", "gate", "post", "pre")


@pytest.mark.parametrize("c,lmax,rows,one_large", [(1, 0, 7, False), (1, 0, 7, True), (5, 1, 6, True), (70, 2, 11, False)])
def test_composed_orders_keep_what_cancels(gpu, c, lmax, rows, one_large):
    """Second derivatives with a recorded graph, their derivatives, and cotangents of weight gradients, with a row's
    entries alike and with one that is much larger (a cotangent's part along the row then cancels almost wholly)."""
    from ictc_o3 import gated_residual_norm
    d = _inputs(c, lmax, rows, 17)
    if one_large:
        d["x"][:, -1] = d["block"][:, -1] = 300.0
    out = []
    for device, dtype in ((gpu, torch.float32), ("cpu", torch.float64)):
        t = _leaves(d, device, dtype)
        h, y = gated_residual_norm(*[t[k] for k in NAMES], channels=c, eps=EPS) if dtype == torch.float32 else \
            _block_end(*[t[k] for k in NAMES], c, lmax, 1.0)
        first = torch.autograd.grad([h, y], [t[k] for k in NAMES], [t["dh"], t["dy"]], create_graph=True)
        second = torch.autograd.grad([first[0], first[1], first[3], first[4]], [t[k] for k in NAMES],
                                     [t["cx"].detach(), t["cb"].detach(), torch.ones_like(first[3]),
                                      torch.ones_like(first[4])], create_graph=True)
        third = torch.autograd.grad([s.square().sum() for s in second], [t[k] for k in NAMES])
        out.append(dict(enumerate([*first, *second, *third])))
    _compare(*out)
