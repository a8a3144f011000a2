"""The registered operators of the blockwise linear and layer norm, as a compiler sees them: no GPU needed."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from float8_experimental_amd import _custom_ops_norm_blockwise as ops

BF16, FP32 = torch.bfloat16, torch.float32


def shapes(outputs):
    return [(tuple(t.shape), t.dtype, t.stride()) for t in outputs]


@pytest.mark.parametrize("k,n", [(128, 256), (100, 130), (64, 256)])
@pytest.mark.parametrize("need_dx", [True, False])
@pytest.mark.parametrize("need_dw", [True, False])
def test_no_tokens_have_the_shapes_that_the_compiler_was_told(k, n, need_dx, need_dw):
    """A batch that is empty (an expert without tokens), forward and backward."""

    def step(b_dtype):
        x, w, b, dy = torch.zeros(0, k, dtype=BF16), torch.zeros(n, k, dtype=FP32), torch.zeros(n, dtype=BF16), torch.zeros(0, n, dtype=BF16)
        y, *saved = ops.blockwise_linear_fwd(x, w, b, need_dx, need_dw)
        return [y, *saved, *ops.blockwise_linear_bwd(dy, *saved, k, FP32, b_dtype, need_dx, need_dw)]

    for b_dtype in (None, BF16, FP32):
        real = step(b_dtype)
        with FakeTensorMode():
            fake = step(b_dtype)
        assert shapes(real) == shapes(fake)
        assert all((t == 0).all() for t in real[6:])
