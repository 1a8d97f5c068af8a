"""The block norms' kernels where a workgroup goes on from row to row, at the widest rows, and the composed orders
behind them, against plain float64 formulas (tolerances as in test_norms_gpu.py: 1e-5 of the largest entry)."""
import pytest
import torch

from test_norms_gpu import EPS, _all_orders, _block_end, _compare, _inputs, _leaves, _norm

pytestmark = pytest.mark.gpu

NAMES = ("x", "block", "gate", "post", "pre")


@pytest.mark.parametrize("c,lmax,rows,one_large", [(1, 0, 7, False), (1, 0, 7, True), (5, 1, 6, True),
                                                   (70, 2, 11, False)])
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


# more rows than workgroups leave partial weight gradients (512 to 2,048 of them, by order and row size), so that each
# goes on to further rows: rows that share a wave, of one wave, of two, of four with operands in LDS, of five to
# eight, of more; and the widest rows with every degree
LONG = [(16, 2, 16500), (64, 3, 2500), (70, 2, 1300), (128, 3, 1300), (256, 3, 1100), (300, 1, 1100), (512, 3, 600),
        (600, 1, 1100), (520, 3, 1030), (600, 2, 5), (1024, 3, 5), (1000, 1, 4)]


@pytest.mark.parametrize("c,lmax,rows", LONG)
def test_norm_where_workgroups_go_on(gpu, c, lmax, rows):
    from ictc_o3 import equivariant_norm
    d = _inputs(c, lmax, rows, c + rows)
    d = {"x": d["x"], "block": None, "gate": None, "post": None, "pre": d["pre"], "dy": d["dy"], "cx": d["cx"]}
    t, ref = _leaves(d, gpu, torch.float32), _leaves(d, "cpu", torch.float64)
    _compare(_all_orders(t, None, equivariant_norm(t["x"], t["pre"], channels=c, eps=EPS)),
             _all_orders(ref, None, _norm(ref["x"], ref["pre"], c, lmax)))


@pytest.mark.parametrize("behind", [True, False])
@pytest.mark.parametrize("c,lmax,rows", LONG)
def test_block_end_where_workgroups_go_on(gpu, c, lmax, rows, behind):
    from ictc_o3 import gated_residual_norm
    d = _inputs(c, lmax, rows, 10 * c + rows, behind=behind)
    t, ref = _leaves(d, gpu, torch.float32), _leaves(d, "cpu", torch.float64)
    got = gated_residual_norm(*[t[k] for k in NAMES], channels=c, residual_scale=0.7, eps=EPS)
    want = _block_end(*[ref[k] for k in NAMES], c, lmax, 0.7)
    _compare(_all_orders(t, *got), _all_orders(ref, *want))


def test_calls_that_ask_the_engine(gpu, monkeypatch):
    """Large calls ask whether weight gradients run: a force loss's gradients (the first ones without the weights'),
    weights alone, and one weight of two."""
    from ictc_o3 import gated_residual_norm
    from ictc_o3.backends.hip import norms
    monkeypatch.setattr(norms, "ASK_FROM", 0)
    c, lmax, rows = 48, 2, 60
    d = _inputs(c, lmax, rows, 21)
    results = []
    for device, dtype in ((gpu, torch.float32), ("cpu", torch.float64)):
        t = _leaves(d, device, dtype)

        def values():
            if dtype == torch.float32:
                return gated_residual_norm(*[t[k] for k in NAMES], channels=c, eps=EPS)
            return _block_end(*[t[k] for k in NAMES], c, lmax, 1.0)

        h, y = values()
        first = torch.autograd.grad([h, y], [t["x"], t["block"]], [t["dh"], t["dy"]], create_graph=True)
        loss = sum(((g - k.detach()) ** 2).sum() for g, k in zip(first, (t["cx"], t["cb"]))) + (y * t["dy"]).sum()
        loss.backward(inputs=[t["post"], t["pre"], t["gate"]])
        out = [*first, t["post"].grad, t["pre"].grad, t["gate"].grad]
        for names in (("post", "pre"), ("pre",), ("post", "x"), ("block",)):
            h, y = values()
            out += torch.autograd.grad([h, y], [t[k] for k in names], [t["dh"].detach(), t["dy"].detach()])
        h, y = values()
        ((h * t["dh"]).sum() + (y * t["dy"]).sum()).backward()
        results.append(dict(enumerate([*out, *[t[k].grad for k in (*NAMES, "dh", "dy")]])))
    _compare(*results)
