"""Layer norm of rows whose size is near the ends of fp32's range, where a product of a number and zero may be no number."""
import pytest
import torch

pytestmark = pytest.mark.gpu
FP = 2.0**-24  # a rounding of fp32


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


@pytest.mark.parametrize("cols", [300, 513, 1030, 2060, 4099, 5000, 8200])
@pytest.mark.parametrize("mean", [1e20, -1e21])
def test_means_whose_square_overflows(f8, cols, mean):
    """Rows about a mean whose square no fp32 holds, with a spread whose square it does.  Some waves of the lanes of such a row hold none of it."""
    x = (mean + 1e17 * torch.randn(5, cols, generator=torch.Generator().manual_seed(cols), dtype=torch.float64)).float().cuda()
    v = x.double()
    rstd = 1 / (v.var(1, keepdim=True, correction=0) + 1e-5).sqrt()
    want = (v - v.mean(1, keepdim=True)) * rstd
    got = f8.layer_norm(x, cols).double()
    # 96 roundings in the mean, which the spread divides, as many in the spread
    tol = 2 * 96 * FP * (v.abs().mean(1, keepdim=True) * rstd + want.abs()) + 4 * FP * v.abs() * rstd
    assert got.isfinite().all() and ((got - want).abs() <= tol).all()
