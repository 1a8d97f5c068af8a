"""What the layers and orthogonalised updates ask for and refuse, without a GPU: workspaces that do not grow with what
a call could be split by, and numbers that are none."""
import ctypes

import pytest
import torch


def _lib():
    from ictc_o3 import _lib as binding
    return binding.lib()


def _muon_workspace(*shapes):
    n = len(shapes)
    return _lib().ictc_hip_muon_workspace(*[(ctypes.c_int64 * n)(*column) for column in zip(*shapes)], n)


@pytest.mark.parametrize("rows,cols", [(8, 8), (64, 64), (1, 5000), (128, 300), (200, 300)])
def test_workspace_of_a_stack_is_bounded(rows, cols):
    """A stack's matrices go through the workspace in groups: 2 GiB of values, and the tables beside them, 1 % of that."""
    at_once, most = _muon_workspace((rows, cols, 1)), 2 ** 31 * 1.02
    assert 0 < at_once < 2 ** 26
    for matrices in (100_000, (1 << 23) - 1, 1 << 23):
        assert at_once < _muon_workspace((rows, cols, matrices)) <= most
    # beside other tensors, and with empty ones between
    assert 0 < _muon_workspace((5, 7, 3), (rows, cols, 1 << 20), (0, 4, 2), (rows, cols, 1 << 20), (700, 600, 2)) <= most


@pytest.mark.parametrize("rows", [1, 2, 100, 254, 255, 256, 1000])
@pytest.mark.parametrize("width", [1, 4, 63, 64, 65, 128, 256, 1000, 1024, 4096])
def test_workspace_of_a_table_gradient_is_bounded(rows, width):
    """Parts of rows stay within 64 MiB or about half of the gradient's size (255 of 512 tokens may be of different rows),
    beside what goes by tokens (keys and places twice, counts) and rows (spans) alone."""
    for count in (1, 2048, 20_000, 65_536, 300_000, 4_000_000, 100_000_000):
        units = _lib().ictc_hip_embedding_workspace(rows, width, count)
        assert 0 < units <= max(2 ** 24, 0.52 * count * width) + 5 * count + 3 * rows + 4096, (count, units)


def test_integers_beyond_a_double_are_refused():
    """As what they are, with nothing pending behind the refusal."""
    from ictc_o3 import embedding, layer_norm
    for large in (10 ** 400, -10 ** 400):
        with pytest.raises(ValueError, match="scale must be a finite number"):
            embedding(torch.zeros(2, dtype=torch.int64), torch.ones(3, 4), scale=large)
        with pytest.raises(ValueError, match="eps must be a positive number"):
            layer_norm(torch.ones(2, 4), torch.ones(4), eps=large)


@pytest.mark.parametrize("scale", [1e39, -1e300, 2 ** 128])
def test_scales_beyond_float32_are_refused(scale):
    """The kernels take the scale as a float32: one that is none there would give infinities for every token."""
    from ictc_o3 import embedding, layer_norm
    with pytest.raises(ValueError, match="scale must be a finite number"):
        embedding(torch.zeros(2, dtype=torch.int64), torch.ones(3, 4), scale=scale)
    with pytest.raises(ValueError, match="eps must be a positive number"):
        layer_norm(torch.ones(2, 4), torch.ones(4), eps=abs(scale))
