"""The registered operators of the blockwise linear and layer norm, as a compiler sees them: no GPU needed."""
import inspect

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import float8_experimental_amd as f8
from float8_experimental_amd import _custom_ops_norm_blockwise as ops
from float8_experimental_amd import _native

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


def test_compiled_layer_norm_computes_what_is_asked_for(monkeypatch):
    """The kernels are stood in for: only which gradients they are asked for is looked at."""
    asked = []

    def backward(dy, x, weight, p_dtype, stats, need_dx=True, need_dw=True, need_db=True):
        asked.append((need_dx, need_dw, need_db))
        return tuple(torch.zeros(s, dtype=d) if need else None for s, d, need in ((x.shape, x.dtype, need_dx), ((x.shape[1],), p_dtype, need_dw), ((x.shape[1],), p_dtype, need_db)))

    monkeypatch.setattr(_native, "layer_norm", lambda x, w, b, eps: (torch.zeros_like(x), torch.zeros(x.shape[0], 2)))
    monkeypatch.setattr(_native, "layer_norm_backward", backward)
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 1, 1)):
        x, w, b = (torch.ones(s, dtype=BF16, requires_grad=bool(r)) for s, r in zip(((3, 8), (8,), (8,)), which))
        ops.layer_norm(x, w, b, 8, 1e-5).sum().backward()
        assert asked.pop() == tuple(map(bool, which)) and not asked
        assert [t.grad is not None for t in (x, w, b)] == list(map(bool, which))
        stats = torch.zeros(3, 2)
        real = ops.layer_norm_bwd(x.detach(), x.detach(), w.detach(), BF16, stats, *map(bool, which))
        with FakeTensorMode(allow_non_fake_inputs=True):
            fake = ops.layer_norm_bwd(x.detach(), x.detach(), w.detach(), BF16, stats, *map(bool, which))
        assert shapes(real) == shapes(fake)
        asked.clear()


def test_clip_grad_norm_takes_the_arguments_of_torch():
    assert list(inspect.signature(f8.clip_grad_norm_).parameters) == list(inspect.signature(torch.nn.utils.clip_grad_norm_).parameters)
