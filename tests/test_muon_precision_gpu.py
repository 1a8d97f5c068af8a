"""Orthogonalised matrices' errors beside those of the same iteration in plain float32 on the CPU, against float64: the
comparison by which lost bits are seen, at random and at rank-deficient matrices, whose null directions' errors grow
485-fold.

Bound.  In units of 2^-24, root mean squares over a value's mantissa: float32 rounds each factor of a product by 0.41,
0.58 for both.  Two float16 parts round it 1.5 times as coarsely (2^-23 in the upper half of lo's range, float32's and finer
below), 0.62, 0.87 for both, and the product of the low parts that is left out is 0.64 of it: 1.08 together, 1.9 times
float32's if the sums were exact.  What float32 sums add, which both have, brings the ratio nearer to 1.  So 2; each
lost bit of the values would double what the parts give, and the low part as a whole is 2^11 of it."""
import pytest
import torch

from test_muon_gpu import COEFFICIENTS

pytestmark = pytest.mark.gpu


def _iterate(u, dtype):
    a, b, c = COEFFICIENTS
    x = (u.double() / (u.double().norm() + 1e-7)).to(dtype)
    turned = x.shape[0] > x.shape[1]
    x = x.mT.contiguous() if turned else x
    for _ in range(5):
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    return (x.mT if turned else x).double()


@pytest.mark.parametrize("rows,columns,rank", [
    (64, 64, 64), (128, 700, 128), (300, 257, 257), (513, 511, 511), (40, 2000, 40), (1024, 200, 200), (64, 64, 16),
    (128, 128, 32), (300, 300, 60), (600, 520, 100), (512, 512, 32), (2, 40, 2), (64, 8, 8), (30, 30, 5)])
def test_errors_beside_float32(gpu, rows, columns, rank):
    from ictc_o3.operators import orthogonalize
    own = plain = 0.0
    for seed in range(6):
        g = torch.Generator().manual_seed(seed)
        u = torch.randn(rows, columns, generator=g)
        if rank < min(rows, columns):
            u = torch.randn(rows, rank, generator=g) @ torch.randn(rank, columns, generator=g)
        want = _iterate(u, torch.float64)
        size = want.square().sum().item()
        own += (orthogonalize([u.to(gpu)])[0].double().cpu() - want).square().sum().item() / size
        plain += (_iterate(u, torch.float32) - want).square().sum().item() / size
    print(f"{rows} x {columns} of rank {rank}: {(own / 6) ** 0.5:.2e}, float32 {(plain / 6) ** 0.5:.2e}, ratio {(own / plain) ** 0.5:.2f}")
    assert own <= 4.0 * plain, (own / plain) ** 0.5
