"""Embedding against plain float64 indexing on the CPU: lookups, the table's gradient (rows of one token, of a
tenth of all, of none, runs across chunks and tiles, tables of one to three sort passes), the adjoint's
adjoint, tokens outside the table, odd widths, graphs, streams and refusals.

Tolerances: a lookup rounds once (2^-24).  A row's sum adds up to 32 terms (or a chunk's, 64 at most) in float32
before sums in 64 bits: 64 u of the sum of magnitudes (u = 6e-8), 4e-6 where they do not cancel; they are
compared with that sum, |dy| summed, as the scale.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

# tokens, rows, width: one, fewer than a chunk, a chunk's borders, a tile and its borders; 8, 9, 16 and 17 bits of
# keys (the largest key is the number of rows); widths of one, odd, several workgroups
SHAPES = [(1, 1, 1), (5, 3, 7), (31, 4, 64), (32, 4, 64), (33, 1, 128), (64, 2, 3), (2047, 10, 128), (2048, 255, 16),
          (2049, 256, 20), (5000, 2, 64), (10000, 100, 65), (30000, 7921, 64), (3, 70000, 33), (4096, 65535, 12),
          (4097, 65536, 12), (50001, 9, 8), (700, 50, 257), (300, 40, 1000), (20000, 1, 256)]


def _case(count, rows, width, seed, dtype=torch.int64, skew=1.0):
    g = torch.Generator().manual_seed(seed)
    weight = torch.arange(1, rows + 1, dtype=torch.float64).pow(-skew)[torch.randperm(rows, generator=g)]
    tokens = torch.multinomial(weight, count, replacement=True, generator=g).to(dtype)
    return tokens, torch.randn(rows, width, generator=g), torch.randn(count, width, generator=g)


def _gradient(tokens, dy, rows, scale):
    keep = (tokens >= 0) & (tokens < rows)
    index, dy = tokens[keep].long(), dy[keep].double()
    zero = torch.zeros(rows, dy.shape[1], dtype=torch.float64)
    return zero.index_add(0, index, dy) * scale, zero.index_add(0, index, dy.abs()) * abs(scale)


def _check_gradient(got, tokens, dy, rows, scale):
    want, size = _gradient(tokens, dy, rows, scale)
    error = (got.double().cpu() - want).abs()
    assert got.shape == want.shape and bool((error <= 4e-6 * size).all()), (error / size.clamp(min=1e-30)).max()


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("count,rows,width", SHAPES)
def test_lookup_and_gradient(gpu, count, rows, width, dtype):
    from ictc_o3.operators import embedding
    tokens, table, dy = _case(count, rows, width, count + rows, dtype)
    leaf = table.to(gpu).requires_grad_()
    y = embedding(tokens.to(gpu), leaf, scale=-0.75)
    assert torch.equal(y.detach().cpu(), table[tokens.long()] * -0.75)
    got, = torch.autograd.grad(y, leaf, dy.to(gpu))
    _check_gradient(got, tokens, dy, rows, -0.75)


@pytest.mark.parametrize("skew", [0.0, 3.0])
def test_even_and_steep_distributions(gpu, skew):
    from ictc_o3.operators import embedding
    tokens, table, dy = _case(40000, 500, 32, 7, skew=skew)
    leaf = table.to(gpu).requires_grad_()
    got, = torch.autograd.grad(embedding(tokens.to(gpu), leaf), leaf, dy.to(gpu))
    _check_gradient(got, tokens, dy, 500, 1.0)


@pytest.mark.parametrize("order", ["sorted", "falling", "alternating", "same"])
def test_given_orders(gpu, order):
    from ictc_o3.operators import embedding
    count, rows = 9001, 300
    tokens, table, dy = _case(count, rows, 48, 8)
    tokens = {"sorted": tokens.sort()[0], "falling": tokens.sort(descending=True)[0],
              "alternating": torch.arange(count) % 2 * (rows - 1), "same": torch.full((count,), rows - 1)}[order]
    leaf = table.to(gpu).requires_grad_()
    got, = torch.autograd.grad(embedding(tokens.to(gpu), leaf), leaf, dy.to(gpu))
    _check_gradient(got, tokens, dy, rows, 1.0)


def test_tokens_outside_the_table(gpu):
    """A padded batch: rows of zeros, no gradient, not-a-number in their cotangents left out; also every token."""
    from ictc_o3.operators import embedding
    tokens, table, dy = _case(3000, 20, 36, 9)
    tokens[::7], tokens[5::11], tokens[3], tokens[4] = -1, 20, 1 << 40, -(1 << 40)
    out = (tokens < 0) | (tokens >= 20)
    dy[out] = float("nan")
    leaf = table.to(gpu).requires_grad_()
    y = embedding(tokens.to(gpu), leaf, scale=2.0)
    assert not y[out.to(gpu)].any() and torch.equal(y.detach().cpu()[~out], table[tokens[~out]] * 2.0)
    got, = torch.autograd.grad(y, leaf, dy.to(gpu))
    _check_gradient(got, tokens, dy, 20, 2.0)
    nowhere = torch.full((100,), -1, device=gpu)
    got, = torch.autograd.grad(embedding(nowhere, leaf), leaf, torch.ones(100, 36, device=gpu))
    assert not got.any()


def test_orders_beyond_the_first(gpu):
    """The gradient of the table's gradient is a lookup, and that one's a table's gradient again."""
    from ictc_o3.operators import embedding
    tokens, table, dy = _case(400, 12, 24, 10)
    at = tokens.to(gpu)
    leaf, top = table.to(gpu).requires_grad_(), dy.to(gpu).requires_grad_()
    first, = torch.autograd.grad(embedding(at, leaf, scale=3.0), leaf, top, create_graph=True)
    cot = torch.randn(12, 24, generator=torch.Generator().manual_seed(1)).to(gpu).requires_grad_()
    second, = torch.autograd.grad(first, top, cot, create_graph=True)
    assert torch.equal(second.detach(), cot.detach()[at] * 3.0)
    third, = torch.autograd.grad(second, cot, dy.to(gpu))
    assert torch.equal(third, first.detach())
    # against differences: the map is linear, so a step of 1 is exact up to rounding
    v = torch.randn(12, 24, generator=torch.Generator().manual_seed(2)).to(gpu)
    with torch.no_grad():
        change = ((embedding(at, leaf + v, scale=3.0) - embedding(at, leaf, scale=3.0)).double() * top.double()).sum()
    assert (first.detach().double() * v.double()).sum().item() == pytest.approx(change.item(), rel=1e-5, abs=1e-3)


def test_shapes_strides_and_alignment(gpu):
    from ictc_o3.operators import embedding
    tokens, table, _ = _case(60, 9, 31, 11)
    flat = torch.randn(9 * 31 + 1, device=gpu)
    odd = flat[1:].view(9, 31)
    at = tokens.view(3, 4, 5).to(gpu)
    assert torch.equal(embedding(at, odd), odd[at])
    assert torch.equal(embedding(at.permute(2, 0, 1), odd.t().contiguous().t()), odd[at.permute(2, 0, 1)])
    assert embedding(at[0, 0, 0], odd).shape == (31,) and embedding(at[:0], odd).shape == (0, 4, 5, 31)
    leaf = table.to(gpu).requires_grad_()
    got, = torch.autograd.grad(embedding(at[:0], leaf), leaf, torch.empty(0, 4, 5, 31, device=gpu))
    assert got.shape == leaf.shape and not got.any()
    got, = torch.autograd.grad(embedding(at, leaf), leaf, torch.ones(1, device=gpu).expand(3, 4, 5, 31))
    _check_gradient(got, tokens, torch.ones(60, 31), 9, 1.0)


def test_runs_agree_in_bits_and_on_another_stream(gpu):
    from ictc_o3.operators import embedding
    tokens, table, dy = (t.to(gpu) for t in _case(60000, 200, 64, 12))
    leaf = table.requires_grad_()
    results = []
    for k in range(2):
        stream = torch.cuda.Stream() if k else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            results.append(torch.autograd.grad(embedding(tokens, leaf), leaf, dy)[0])
        torch.cuda.synchronize()
    assert torch.equal(*results)


def test_captured_passes(gpu):
    """Lookup and gradient in a graph, replayed on new tokens and cotangents between eager calls."""
    from ictc_o3.operators import embedding

    def work(tokens, table, dy):
        leaf = table.detach().requires_grad_()
        y = embedding(tokens, leaf, scale=1.5)
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]

    static = [t.to(gpu) for t in _case(5000, 300, 40, 13)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(*static)
    for seed in range(3):
        for old, new in zip(static, _case(5000, 300, 40, 50 + seed, skew=float(seed))):
            old.copy_(new)
        graph.replay()
        want = work(*[t.clone() for t in static])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_a_large_table(gpu):
    """Rows beyond 2^31 bytes and values: offsets are 64 bits wide."""
    from ictc_o3.operators import embedding
    rows, width = 2_200_000, 1001
    table = torch.zeros(rows, width, device=gpu)
    tokens = torch.tensor([rows - 1, 5, rows - 1, 0], device=gpu)
    table[rows - 1] = torch.arange(width, device=gpu)
    leaf = table.requires_grad_()
    y = embedding(tokens, leaf)
    assert torch.equal(y[0].detach(), torch.arange(width, device=gpu).float()) and not y[1].any()
    got, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert bool((got[rows - 1] == 2).all()) and bool((got[5] == 1).all()) and bool((got[0] == 1).all())
    got[[rows - 1, 5, 0]] = 0
    assert not got.any()


def test_refusals(gpu):
    from ictc_o3.operators import embedding
    tokens, table = torch.zeros(4, dtype=torch.int64, device=gpu), torch.zeros(3, 8, device=gpu)
    for call in (lambda: embedding(tokens.float(), table), lambda: embedding(tokens.short(), table),
                 lambda: embedding(tokens.cpu(), table), lambda: embedding(tokens, table[0]),
                 lambda: embedding(tokens, table[:0]), lambda: embedding(tokens, table[:, :0]),
                 lambda: embedding(tokens, table.double()), lambda: embedding(tokens, table, scale=float("nan")),
                 lambda: embedding(tokens, table, scale="1"), lambda: embedding(tokens, table, scale=True)):
        with pytest.raises(ValueError):
            call()


def test_inference_and_changed_tokens(gpu):
    from ictc_o3.operators import embedding
    tokens, table, dy = (t.to(gpu) for t in _case(50, 6, 16, 14))
    with torch.inference_mode():
        assert torch.equal(embedding(tokens, table, scale=2.0), table[tokens] * 2.0)
    leaf = table.requires_grad_()
    y = embedding(tokens, leaf)
    tokens.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, leaf, dy)


def test_two_streams_at_once(gpu):
    from ictc_o3.operators import embedding
    cases = [tuple(t.to(gpu) for t in _case(60000, rows, 64, rows)) for rows in (90, 4000)]
    leaves = [c[1].requires_grad_() for c in cases]
    work = lambda c, leaf: torch.autograd.grad(embedding(c[0], leaf), leaf, c[2])[0]     # noqa: E731
    want = [work(c, leaf).clone() for c, leaf in zip(cases, leaves)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, c, leaf in zip(streams, cases, leaves):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(work(c, leaf))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
