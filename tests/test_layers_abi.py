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
    from ictc_o3 import layer_norm
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(2, 8), torch.ones(8))
