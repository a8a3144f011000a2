"""The gradient of a bias has the precision of the bias: an fp32 one beside 16-bit activations is not rounded to theirs."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("compiled", [False, True])
@pytest.mark.parametrize("dtype,b_dtype", [(BF16, FP32), (FP16, FP32), (BF16, BF16), (FP32, BF16), (BF16, FP16), (FP32, FP32)])
def test_one_rounding(dtype, b_dtype, compiled):
    """Whole numbers: every sum in fp32 is exact, so that the rounding to the type of the bias is the only one."""
    import float8_experimental_amd as f8

    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(1000, 136, generator=g).to(dtype).cuda(), torch.randn(200, 136, generator=g).to(dtype).cuda()
    b, dy = torch.zeros(200, dtype=b_dtype, device="cuda", requires_grad=True), torch.randint(0, 17, (1000, 200), generator=g).to(dtype).cuda()
    linear = torch.compile(f8.blockwise_linear, fullgraph=True) if compiled else f8.blockwise_linear
    linear(x, w, b).backward(dy)
    assert b.grad.dtype == b_dtype and torch.equal(b.grad, dy.double().sum(0).to(b_dtype))
