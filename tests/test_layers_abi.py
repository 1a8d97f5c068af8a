"""The layers' C entry points without a GPU: what is not valid is refused before any launch, and nothing to do
launches nothing."""
import ctypes

import pytest
import torch

F = ctypes.c_void_p(256)     # an address that no call below gets as far as using


def _lib():
    from ictc_o3 import _lib as binding
    return binding.lib()


def test_layer_norm_arguments():
    lib = _lib()
    ws = lib.ictc_hip_layer_norm_workspace(64, 100)
    assert ws > 0 and lib.ictc_hip_layer_norm_workspace(64, 0) > 0
    forward, backward, second = (lib.ictc_hip_layer_norm_forward, lib.ictc_hip_layer_norm_backward,
                                 lib.ictc_hip_layer_norm_second)
    assert forward(F, F, F, F, 64, 1, 1e-5, 0, None) == 0
    for width, activation, eps, rows in ((0, 0, 1e-5, 4), (8193, 0, 1e-5, 4), (64, 2, 1e-5, 4), (64, -1, 1e-5, 4),
                                         (64, 0, 0.0, 4), (64, 0, float("nan"), 4), (64, 0, float("inf"), 4),
                                         (64, 0, 1e-5, -1)):
        assert forward(F, F, F, F, width, activation, eps, rows, None) == 1
        assert backward(F, F, F, F, F, None, None, None, 0, width, activation, eps, rows, None) == 1
        assert second(F, F, F, F, F, F, F, None, None, None, 0, width, activation, eps, rows, None) == 1
    assert lib.ictc_hip_layer_norm_workspace(0, 4) == -1 and lib.ictc_hip_layer_norm_workspace(64, -1) == -1
    for k in (0, 1, 3):
        args = [F] * 4
        args[k] = None
        assert forward(*args, 64, 0, 1e-5, 4, None) == 1
    assert backward(F, F, F, F, F, F, F, F, ws - 1, 64, 0, 1e-5, 100, None) == 1
    assert backward(F, F, F, F, F, F, F, None, ws, 64, 0, 1e-5, 100, None) == 1
    assert backward(F, F, F, None, F, None, None, None, 0, 64, 0, 1e-5, 100, None) == 1
    assert backward(F, F, F, F, None, None, None, None, 0, 64, 0, 1e-5, 100, None) == 0      # nothing asked for
    assert second(F, F, F, F, None, F, F, None, None, None, 0, 64, 0, 1e-5, 100, None) == 1
    assert second(F, F, F, F, F, F, F, F, F, F, ws - 1, 64, 0, 1e-5, 100, None) == 1
    assert second(F, F, F, F, F, None, None, None, None, None, 0, 64, 0, 1e-5, 100, None) == 0


def test_python_guards_refuse_cpu_tensors():
    from ictc_o3 import embedding, layer_norm, muon_step, orthogonalize
    from ictc_o3.optim import Muon
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(2, 8), torch.ones(8))
    with pytest.raises(ValueError):
        embedding(torch.zeros(2, dtype=torch.int64), torch.ones(8, 4))
    x = torch.zeros(4, 4)
    for call in (lambda: orthogonalize([x]), lambda: muon_step([x], [x], [x], lr=0.1)):
        with pytest.raises(ValueError):
            call()
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(eps=0.0), dict(weight_decay=-1.0), dict(ns_steps=0),
                dict(ns_coefficients=(1.0, 2.0)), dict(adjust_lr_fn="none"), dict(max_grad_norm=0.0)):
        with pytest.raises(ValueError):
            Muon([torch.nn.Parameter(x)], **bad)
    for params in ([torch.nn.Parameter(x[0])], [torch.nn.Parameter(x[:, :2])]):
        with pytest.raises(ValueError):
            Muon(params)


def test_embedding_arguments():
    lib = _lib()
    forward, gradient = lib.ictc_hip_embedding_forward, lib.ictc_hip_embedding_table_grad
    units = lib.ictc_hip_embedding_workspace(10, 64, 1000)
    assert units > 0 and lib.ictc_hip_embedding_workspace(10, 64, 100000) > units
    assert forward(F, 8, F, F, 10, 64, 1.0, 0, None) == 0
    for width_of_index, rows, width, count in ((2, 10, 64, 4), (8, 0, 64, 4), (8, 1 << 31, 64, 4), (8, 10, 0, 4),
                                               (8, 10, (1 << 20) + 1, 4), (8, 10, 64, -1), (4, 10, 64, 1 << 31)):
        assert forward(F, width_of_index, F, F, rows, width, 1.0, count, None) == 1
        assert gradient(F, width_of_index, F, F, rows, width, 1.0, count, F, 1 << 60, None) == 1
    assert lib.ictc_hip_embedding_workspace(0, 64, 4) == -1
    for k in (0, 2, 3):
        args = [F, 8, F, F]
        args[k] = None
        assert forward(*args, 10, 64, 1.0, 4, None) == 1
        assert gradient(*args, 10, 64, 1.0, 1000, F, units, None) == 1
    assert gradient(F, 8, F, F, 10, 64, 1.0, 1000, F, units - 1, None) == 1
    assert gradient(F, 8, F, F, 10, 64, 1.0, 1000, None, units, None) == 1
    assert gradient(F, 8, F, F, 10, 64, 1.0, 1000, ctypes.c_void_p(260), units, None) == 1
    assert gradient(F, 8, F, F, 10, 64, 1.0, 0, F, units, None) == 1


def _arrays(*shapes):
    n = len(shapes)
    return [(ctypes.c_int64 * n)(*column) for column in zip(*shapes)], (ctypes.c_void_p * n)(*[256] * n), n


def test_muon_arguments():
    from ictc_o3 import _lib as binding
    lib = _lib()
    good = dict(beta=0.95, weight_decay=0.0, eps=1e-7, coefficients=(ctypes.c_double * 3)(3.4, -4.7, 2.0), lr=0.1,
                nesterov=1, steps=5, adjust=0)
    make = lambda **more: ctypes.byref(binding.MuonDesc(**{**good, **more}))     # noqa: E731
    shapes, at, n = _arrays((64, 64, 1), (10, 300, 3))
    need = lib.ictc_hip_muon_workspace(*shapes, n)
    assert need > 0 and lib.ictc_hip_muon_workspace(*_arrays((64, 64, 0), (0, 5, 1))[0], 2) == 0
    assert lib.ictc_hip_muon_workspace(*shapes, -1) == -1 and lib.ictc_hip_muon_workspace(None, *shapes[1:], n) == -1
    for shape in ((-1, 64, 1), (64, -1, 1), (64, 64, -1), ((1 << 20) + 1, 64, 1), (64, 64, 1 << 24),
                  (1 << 20, 1 << 20, 1)):
        assert lib.ictc_hip_muon_workspace(*_arrays(shape)[0], 1) == -1, shape

    def orthogonalize(desc, src=at, out=at, shapes=shapes, count=n, ws=F, size=need):
        return lib.ictc_hip_orthogonalize(src, out, *shapes, count, desc, ws, size, None)

    def step(desc, p=at, g=at, m=at, shapes=shapes, count=n, ws=F, size=need):
        return lib.ictc_hip_muon_step(p, g, m, *shapes, count, desc, None, None, ws, size, None)

    none = (ctypes.c_void_p * 2)(None, None)
    for call in (orthogonalize, step):
        assert call(make(), count=0) == 0
        assert call(make(), shapes=_arrays((64, 64, 0), (0, 5, 1))[0]) == 0      # no values
        assert call(None) == 1 and call(make(), count=-1) == 1
        for bad in (dict(beta=1.0), dict(beta=float("nan")), dict(weight_decay=-1.0), dict(eps=0.0), dict(steps=0),
                    dict(eps=float("inf")), dict(steps=65), dict(adjust=2), dict(lr=-1.0), dict(lr=float("nan")),
                    dict(coefficients=(ctypes.c_double * 3)(1.0, float("nan"), 0.0))):
            assert call(make(**bad)) == 1, bad
        assert call(make(), ws=None) == 1 and call(make(), size=need - 1) == 1
        assert call(make(), ws=ctypes.c_void_p(264)) == 1
    assert orthogonalize(make(), src=None) == 1 and orthogonalize(make(), out=none) == 1
    assert orthogonalize(make(), src=none) == 1
    assert step(make(), p=none) == 1 and step(make(), m=none) == 1 and step(make(), g=None) == 1
    assert step(make(), g=none) == 0                                             # no tensor takes part
