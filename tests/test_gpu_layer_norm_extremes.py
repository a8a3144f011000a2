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


# (columns, log2 of the values, eps): the sum of a row is finite, a value times 1 / sqrt(eps) is not
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols,log2,eps", [(8, 120, 1e-5), (64, 121, 1e-5), (128, 113, 1e-12), (20001, 112, 1e-12)])
def test_gradients_of_constant_rows_of_large_values(f8, cols, log2, eps, dtype):
    """Their mean is exact and their variance zero: xhat is zero and dx is (dy - mean(dy)) / sqrt(eps), in rows that end inside a lane's piece too."""
    x = torch.full((3, cols), 2.0**log2, dtype=dtype, device="cuda", requires_grad=True)
    w = torch.ones(cols, dtype=dtype, device="cuda", requires_grad=True)
    dy = (torch.randn(3, cols, generator=torch.Generator().manual_seed(cols)) * 2.0**-10).to(dtype).cuda()
    f8.layer_norm(x, cols, w, eps=eps).backward(dy)
    d = dy.double()
    want = (d - d.mean(1, keepdim=True)) / eps**0.5
    # one rounding to the output's type, and sums of 96 roundings
    tol = (2.0**-8 if dtype is torch.bfloat16 else 2.0**-23) * want.abs() + 96 * FP * (d.abs() + d.abs().mean(1, keepdim=True)) / eps**0.5
    assert ((x.grad.double() - want).abs() <= tol).all() and (w.grad == 0).all()


@pytest.mark.parametrize("cols", [7, 63, 109, 379, 500, 731, 1000, 2035, 4093])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_constant_rows_have_no_variance(f8, cols, dtype):
    """Eight significant bits, so that every sum is exact: the mean is the value itself, and not an ulp beside it (whose square is 1.5e-5, more than eps)."""
    x = torch.full((3, cols), 98816.0, dtype=dtype, device="cuda", requires_grad=True)
    b = torch.randn(cols, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    dy = torch.randn(3, cols, generator=torch.Generator().manual_seed(cols)).to(dtype).cuda()
    y = f8.layer_norm(x, cols, None, b)
    assert torch.equal(y, b.expand(3, cols))
    y.backward(dy)
    d = dy.double()
    want = (d - d.mean(1, keepdim=True)) / 1e-5**0.5
    tol = (2.0**-8 if dtype is torch.bfloat16 else 2.0**-23) * want.abs() + 96 * FP * (d.abs() + d.abs().mean(1, keepdim=True)) / 1e-5**0.5
    assert ((x.grad.double() - want).abs() <= tol).all()
