"""The optimizer's and the norms' C entry points and the host module without a GPU: what is not valid is
refused before any launch, and nothing to do launches nothing."""
import ctypes

import pytest
import torch

F = ctypes.c_void_p(256)     # an address that no call below gets as far as using


def _lib():
    from ictc_o3 import _lib as binding
    return binding, binding.lib()


def _arrays(*sizes):
    n = len(sizes)
    return (ctypes.c_void_p * n)(*[256] * n), (ctypes.c_int64 * n)(*sizes), n


def test_gradient_norm_arguments():
    _, lib = _lib()
    at, sizes, n = _arrays(10, 20)
    need = lib.ictc_hip_gradient_norm_workspace(n)
    assert need > 0 and lib.ictc_hip_gradient_norm_workspace(10 ** 4) > need
    assert lib.ictc_hip_gradient_norm_workspace(-1) == -1
    call = lib.ictc_hip_gradient_norm
    assert call(at, sizes, -1, 1.0, F, need, F, None) == 1
    assert call(None, sizes, n, 1.0, F, need, F, None) == 1
    assert call(at, sizes, n, 1.0, None, need, F, None) == 1
    assert call(at, sizes, n, 1.0, F, need - 1, F, None) == 1
    assert call(at, sizes, n, 1.0, F, need, None, None) == 1
    assert call(at, sizes, n, float("nan"), F, need, F, None) == 1
    assert call(at, _arrays(10, -1)[1], n, 1.0, F, need, F, None) == 1
    assert call(at, _arrays(10, 1 << 50)[1], n, 1.0, F, need, F, None) == 1
    assert call((ctypes.c_void_p * 2)(256, None), sizes, n, 1.0, F, need, F, None) == 1


def test_adamw_arguments():
    binding, lib = _lib()
    at, sizes, n = _arrays(300, 7)
    call = lib.ictc_hip_adamw_step

    def step(desc, params=at, grads=at, elements=sizes, count=n, m=F, v=F, mt=F, vt=F, progress=F):
        return call(params, grads, elements, count, None if desc is None else ctypes.byref(desc), m, v, mt, vt, progress,
                    None, None, None)

    good = dict(beta1=0.9, beta2=0.999, weight_decay=0.0, lr=1e-3, eps=1e-8, seed=0, moment_bits=32)
    make = lambda **more: binding.AdamwDesc(**{**good, **more})     # noqa: E731
    assert step(make(), count=0) == 0
    none = (ctypes.c_void_p * 2)(None, None)
    assert step(make(), grads=none) == 0                            # no tensor takes part
    assert step(None) == 1
    assert step(make(moment_bits=16)) == 2
    for bad in (dict(beta1=1.0), dict(beta2=-0.1), dict(lr=-1.0), dict(lr=float("nan")), dict(eps=-1.0),
                dict(weight_decay=-1.0), dict(beta1=float("nan"))):
        assert step(make(**bad)) == 1, bad
    assert step(make(), count=-1) == 1
    assert step(make(), params=None) == 1
    assert step(make(), params=none) == 1                           # a gradient without a parameter
    assert step(make(), elements=_arrays(300, -7)[1]) == 1
    assert step(make(), elements=_arrays(300, 1 << 50)[1]) == 1
    assert step(make(), m=None) == 1 and step(make(), progress=None) == 1
    assert step(make(), m=ctypes.c_void_p(260)) == 1                # float moments are read 16 bytes at a time
    assert step(make(moment_bits=8), m=ctypes.c_void_p(258)) == 1
    assert step(make(moment_bits=8), mt=None) == 1
    values = lib.ictc_hip_moment_values
    assert values(F, F, F, F, F, F, 100, None) == 1 and values(F, F, F, F, F, F, -256, None) == 1
    assert values(None, F, F, F, F, F, 256, None) == 1 and values(None, F, F, F, F, F, 0, None) == 0
    assert values(F, F, F, F, ctypes.c_void_p(264), F, 256, None) == 1


def test_norm_arguments():
    binding, lib = _lib()
    good = dict(channels=16, lmax=2, input_lmax=2, residual_scale=1.0, eps=1e-5)
    make = lambda **more: ctypes.byref(binding.NormDesc(**{**good, **more}))     # noqa: E731
    ws = lib.ictc_hip_norm_workspace(make(), 100)
    assert ws > 0
    forward, backward, second = lib.ictc_hip_norm_forward, lib.ictc_hip_norm_backward, lib.ictc_hip_norm_second
    assert forward(make(), F, F, F, F, F, F, F, 0, None) == 0
    for bad in (dict(channels=0), dict(channels=1025), dict(lmax=4), dict(lmax=-1), dict(input_lmax=-1), dict(eps=0.0),
                dict(eps=float("nan"))):
        assert forward(make(**bad), F, F, F, F, F, F, F, 4, None) == 1, bad
        assert lib.ictc_hip_norm_workspace(make(**bad), 4) == -1
    assert forward(make(), F, F, F, F, F, F, F, -1, None) == 1
    assert forward(make(), None, F, F, F, F, F, F, 4, None) == 1
    assert forward(make(), F, F, F, None, F, F, F, 4, None) == 1      # a block without its weight
    assert forward(make(), F, F, F, F, F, None, F, 4, None) == 1
    assert forward(make(), F, F, F, F, F, F, None, 4, None) == 1      # a norm behind without its result
    assert forward(make(), F, None, F, None, F, None, F, 4, None) == 1     # a gate without a block
    assert forward(make(input_lmax=1), F, None, None, None, F, None, F, 4, None) == 1
    assert backward(make(), F, F, F, F, F, F, F, F, F, F, F, F, F, ws - 1, 100, None) == 1
    assert backward(make(), F, F, F, F, F, F, F, F, F, F, F, F, None, ws, 100, None) == 1
    assert backward(make(), F, F, None, F, F, F, F, F, F, F, None, None, None, 0, 100, None) == 1     # gate's gradient
    assert backward(make(), F, F, F, F, None, F, F, F, F, F, None, None, None, 0, 100, None) == 1     # grad_y without pre
    assert backward(make(), F, F, F, F, F, None, None, F, F, F, None, None, None, 0, 100, None) == 1  # no cotangent
    assert second(make(), F, F, F, F, F, F, None, F, F, F, F, F, F, F, None, None, None, None, 0, 100, None) == 1
    assert second(make(), F, F, F, F, F, None, None, F, F, F, None, F, F, F, None, None, None, None, 0, 100, None) == 1
    assert second(make(), F, F, None, F, F, F, F, F, F, F, F, F, None, F, F, None, None, None, 0, 100, None) == 1
    assert second(make(), F, F, F, F, F, F, F, F, F, F, F, F, F, F, F, F, F, F, ws - 1, 100, None) == 1


def test_host_module():
    binding, _ = _lib()
    host = binding.host()
    cpu = torch.zeros(3)
    for call in (lambda: host.addresses([cpu], "gradients"), lambda: host.addresses([None], "gradients"),
                 lambda: host.pairs([cpu], [cpu], 256), lambda: host.pairs([], [], 256),
                 lambda: host.pairs([cpu], [], 256), lambda: host.pairs([1], [None], 256)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        host.addresses((cpu,), "gradients")
    assert host.addresses([], "gradients") == (-1, b"", b"", True)
    before = cpu._version
    host.written([cpu, cpu], [None, cpu])
    assert cpu._version == before + 1


def test_python_guards_refuse_cpu_tensors():
    from ictc_o3 import adamw_step, equivariant_norm, gated_residual_norm, gradient_norm, moment_values
    from ictc_o3.optim import AdamW
    x, w = torch.zeros(2, 16), torch.ones(8)
    for call in (lambda: gradient_norm([x]), lambda: adamw_step([x], [x], x, x, x, lr=1e-3),
                 lambda: equivariant_norm(x, w, channels=4), lambda: gated_residual_norm(x, x, None, w, w, channels=4),
                 lambda: moment_values((x, x), (x, x))):
        with pytest.raises(ValueError):
            call()
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(moment_bits=16),
                dict(max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(x)], **bad)
